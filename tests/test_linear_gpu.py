"""Dense layers and their gradients on the GPU against 64 bits (bounds:
head_cases.py)."""
import pytest
import torch

import head_cases as hc
from expert_cases import DTYPES, gen, padded, randn, within

pytestmark = pytest.mark.gpu
ACTS = ["none", "relu", "elu", "gelu", "silu"]

SIZES = [(1, 1, 1), (1, 4096, 512), (1, 37, 1000), (2, 8, 3), (3, 602, 41), (5, 2048, 2048),
         (8, 1024, 4096), (16, 512, 640), (17, 300, 130), (31, 8192, 256), (33, 64, 64),
         (64, 1000, 70), (130, 257, 129), (200, 96, 1024), (500, 33, 7), (1000, 256, 256),
         (1031, 602, 256), (700, 8, 2000), (2000, 40, 41), (4096, 64, 16), (3000, 512, 520),
         (260, 4096, 264), (2048, 2048, 2048), (5000, 1024, 1280), (40000, 128, 24),
         (4096, 1024, 4096), (8200, 520, 4104), (20, 1500, 900), (32, 40000, 16), (70, 6000, 8)]


def code(tg, name):
    return dict(none=tg.EPI_NONE, relu=tg.EPI_RELU, elu=tg.EPI_ELU, gelu=tg.EPI_GELU,
                silu=tg.EPI_SILU)[name]


def make(m, k, n, dt, transpose, seed=0, scale=1.0):
    g = gen(m + 3 * k + 7 * n + seed)
    return dict(x=randn(g, (m, k), dt, scale),
                w=randn(g, (n, k) if transpose else (k, n), dt, k ** -0.5),
                bias=randn(g, n, dt, 0.3), residual=randn(g, (m, n), dt), dy=randn(g, (m, n), dt))


def check(p, name, transpose, bias=True, residual=True, pad=(0, 0, 0, 0, 0)):
    import tinygnn_amd as tg
    dt = p["x"].dtype
    x, w = padded(p["x"], pad[0]), padded(p["w"], pad[1])
    b, r = p["bias"] if bias else None, padded(p["residual"], pad[2]) if residual else None
    y, pre = tg.linear(x, w, bias=b, epilogue=code(tg, name), residual=r, transpose=transpose,
                       with_pre=True)
    want, tol, v, off = hc.linear(p["x"], p["w"], b, name, p["residual"] if residual else None,
                                  transpose)
    within(y, want, hc.rounded(want, tol, dt), "y")
    within(pre, v, hc.rounded(v, off, dt), "pre")
    same = tg.linear(x, w, bias=b, epilogue=code(tg, name), residual=r, transpose=transpose)
    assert torch.equal(same, y)
    dy, kept = padded(p["dy"], pad[3]), padded(pre, pad[4])
    dx, dw, db = tg.linear_backward(dy, x, w, pre=kept if name != "none" else None,
                                    epilogue=code(tg, name), bias=bias, transpose=transpose)
    ref = hc.linear_backward(p["dy"], p["x"], p["w"], pre, name, transpose, dt)
    assert (db is None) == (not bias)
    for got, key in ((dx, "dx"), (dw, "dw"), (db, "db")):
        if got is not None:
            within(got, ref[key][0], hc.rounded(*ref[key], dt), key)
    return y, dx, dw, db


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(gpu, m, k, n, transpose, dtype):
    name = ACTS[(m + k + n) % 5]
    check(make(m, k, n, DTYPES[dtype], transpose), name, transpose, bias=(m + n) % 3 != 0,
          residual=k % 2 == 0)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("scale", [1.0, 30.0])
def test_activations(gpu, name, dtype, scale):
    check(make(300, 64, 96, DTYPES[dtype], False, scale=scale), name, False)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("pad", [(1, 1, 1, 1, 1), (2, 6, 8, 3, 1), (8, 8, 8, 8, 8)])
def test_strides(gpu, pad, transpose, dtype):
    """Rows apart, with NaN between them."""
    for m, k, n in ((9, 72, 40), (300, 200, 136)):
        check(make(m, k, n, DTYPES[dtype], transpose), "silu", transpose, pad=pad)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n", [(3, 700, 90), (400, 64, 129), (1, 4096, 4096)])
def test_onto_the_residual(gpu, m, k, n, dtype):
    import tinygnn_amd as tg
    p = make(m, k, n, DTYPES[dtype], False)
    want = tg.linear(p["x"], p["w"], residual=p["residual"])
    wide = padded(p["residual"], 4, fill=5.0)
    got = tg.linear(p["x"], p["w"], residual=wide, out=wide)
    assert got.data_ptr() == wide.data_ptr() and torch.equal(got, want)
    assert bool((wide.as_strided((m, 4), wide.stride(), n) == 5.0).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n", [(1, 1, 1024), (15, 127, 1031), (16, 4096, 1024), (16, 4095, 1040),
                                   (7, 2000, 16384), (16, 4100, 1024), (3, 64, 16400)])
def test_few_rows(gpu, m, k, n, dtype):
    """w's rows along the contraction, at the ends of where one launch takes them."""
    p = make(m, k, n, DTYPES[dtype], True)
    check(p, "silu", True)
    check(p, "none", True, bias=False, residual=False, pad=(8, 8, 0, 0, 0))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,n", [(300000, 41), (40000, 4096), (1000, 3)])
def test_long_sums_of_the_bias_gradient(gpu, m, n, dtype):
    """Values of one sign: chains of 64 rows, of 64 such, and trees of as many parts
    leave 256 roundings of the sum at most."""
    import tinygnn_amd as tg
    dt = DTYPES[dtype]
    dy = ((1 + torch.rand(m, n, generator=gen(m), device="cuda")) / 32).to(dt)
    one = torch.ones(m, 1, dtype=dt, device="cuda")
    _, _, db = tg.linear_backward(dy, one, torch.ones(1, n, dtype=dt, device="cuda"), bias=True)
    want = dy.double().sum(0)
    within(db, want, hc.rounded(want, 256 * hc.U * want, dt), "db")


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_nothing_to_contract(gpu, dtype):
    """k = 0: the epilogue of zeros, by tiles."""
    import tinygnn_amd as tg
    dt = DTYPES[dtype]
    p = make(100, 1, 70, dt, False)
    y = tg.linear(p["x"][:, :0], p["w"][:0], bias=p["bias"], residual=p["residual"])
    want = p["residual"].double() + p["bias"].double()
    within(y, want, hc.rounded(want, 2 * hc.U * want.abs(), dt), "y")


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_empty(gpu, dtype):
    import tinygnn_amd as tg
    dt = DTYPES[dtype]

    def z(*shape):
        return torch.ones(*shape, dtype=dt, device="cuda")

    assert tg.linear(z(0, 5), z(5, 3)).shape == (0, 3)
    assert tg.linear(z(4, 5), z(5, 0)).shape == (4, 0)
    b, r = 2 * z(3), z(4, 3)
    assert bool((tg.linear(z(4, 0), z(0, 3), bias=b, residual=r) == 3).all())
    dx, dw, db = tg.linear_backward(z(0, 3), z(0, 5), z(5, 3), bias=True)
    assert dx.shape == (0, 5) and not dw.any() and not db.any() and dw.shape == (5, 3)
    dx, dw, db = tg.linear_backward(z(4, 0), z(4, 5), z(5, 0), bias=True)
    assert dx.shape == (4, 5) and not dx.any() and dw.shape == (5, 0) and db.shape == (0,)
    dx, dw, db = tg.linear_backward(z(4, 3), z(4, 0), z(0, 3), bias=True)
    assert dx.shape == (4, 0) and dw.shape == (0, 3) and bool((db == 4).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_nan_and_infinities_stay_in_their_rows(gpu, dtype):
    """A NaN row of x makes its own row NaN and no other (nor does what lies
    beyond the matrix in its last tile)."""
    import tinygnn_amd as tg
    for m, k, n in ((5, 40, 24), (300, 100, 130), (600, 520, 264)):
        p = make(m, k, n, DTYPES[dtype], False)
        want = tg.linear(p["x"], p["w"], residual=p["residual"])
        p["x"][m // 2] = float("nan")
        got = tg.linear(p["x"], p["w"], residual=p["residual"])
        assert bool(torch.isnan(got[m // 2]).all())
        got[m // 2] = want[m // 2]
        assert torch.equal(got, want)


def test_gradients_by_differences(gpu):
    """Along each gradient's own direction, central differences of the 64-bit
    form: steps of 1e-4 leave 1e-8 of a third derivative, the gradient's own
    rounding 1e-6 of its length."""
    import tinygnn_amd as tg
    for name in ("elu", "gelu", "silu", "none"):
        p = make(50, 30, 20, torch.float32, False)
        _, pre = tg.linear(p["x"], p["w"], bias=p["bias"], epilogue=code(tg, name), with_pre=True)
        dx, dw, db = tg.linear_backward(p["dy"], p["x"], p["w"], pre=pre, epilogue=code(tg, name),
                                        bias=True)

        def loss(x, w, b):
            return (hc.act(x @ w + b, name)[0] * p["dy"].double()).sum()

        base = [p[i].double() for i in ("x", "w", "bias")]
        for i, g in enumerate((dx, dw, db)):
            d = g.double() / g.double().norm()
            ends = []
            for s in (1e-4, -1e-4):
                moved = list(base)
                moved[i] = moved[i] + s * d
                ends.append(loss(*moved))
            want = (ends[0] - ends[1]) / 2e-4
            assert abs(g.double().norm() - want) <= 1e-5 * abs(want) + 1e-6, (name, i)


def test_equal_calls_give_equal_bits(gpu):
    for dt in DTYPES.values():
        p = make(2000, 300, 70, dt, False)
        a, b = (check(p, "gelu", False) for _ in range(2))
        assert all(torch.equal(s, t) for s, t in zip(a, b))
