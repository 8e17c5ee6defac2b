"""Each tile shape of the grouped and e4m3 products, by the kernel that ran,
at sizes from both sides of the rules that choose it, against 64 bits.

Tolerances (u = 2^-24) as in test_grouped_gpu: a float32 sum of k products is
off by (k + 8) u sum|a||b| at most, bias and epilogue among it, the result
rounded to its type; e4m3 products of 16-bit results by 2^-12 sum|a||b| more.
Where operands are -1, 0 and 1 the sums are exact, and results equal."""
import re

import pytest
import torch

from expert_cases import (DTYPES, U, e4m3, gen, grouped, half_step, least, offsets_of, randn,
                          wgrad, within)

pytestmark = pytest.mark.gpu


def kernels(fn):
    """fn's result and the names of the kernels that it ran."""
    from torch.profiler import ProfilerActivity, profile
    with profile(activities=[ProfilerActivity.CUDA], acc_events=True) as p:
        out = fn()
        torch.cuda.synchronize()
    return out, [e.key for e in p.key_averages()]


def ran(names, kernel, shape=None, flags=None):
    """The one kernel of a name ran, with a tile of `shape` and the flags behind
    it.  (Its name is mangled or not, as the profiler can; where that sees no
    kernel at all, nothing is said.)"""
    if not any("_kernel" in n for n in names):
        return
    found = [n for n in names if re.search(rf"(\b|\d){kernel}(<|I)", n)]
    assert len(found) == 1, (kernel, names)
    if shape is not None:
        at = re.search(r"Shape(?:<|ILi)(\d+)(?:, |ELi)(\d+)(.*)", found[0])
        assert (int(at[1]), int(at[2])) == shape, found[0]
        got = [f in ("true", "Lb1E") for f in re.findall(r"true|false|Lb[01]E", at[3])]
        assert flags is None or got == flags, found[0]


def tolerance(want, size, k, dt, own=0.0):
    return ((k + 8) * U * size + half_step(dt) * (want.abs() + (k + 8) * U * size) + least(dt)
            + (1 + half_step(dt)) * own * size)


def fp8_operands(g, m, k, n, e=None):
    """Quantised operands and their values in 64 bits."""
    import tinygnn_amd as tg
    lead = () if e is None else (e,)
    x = randn(g, (m, k), torch.bfloat16)
    w = randn(g, (*lead, k, n), torch.bfloat16, k ** -0.5)
    xq, wq = tg.quantize(x), tg.quantize_weight(w)
    wide = wq.scale.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)
    return xq, wq, e4m3(x)[0], (wq.q.double() * wide)[..., :k].transpose(-1, -2)


def check_fp8(dt, m, k, n, sizes, gather, want_shape):
    import tinygnn_amd as tg
    g = gen(m + k + n)
    xq, wq, xv, wv = fp8_operands(g, m, k, n, None if sizes is None else len(sizes))
    off = rows = None
    many = m
    if gather:
        many = sum(sizes) + 9
        rows = torch.randint(0, m, (many,), generator=g, device="cuda", dtype=torch.int32)
        rows[[3, many // 2]] = torch.tensor([m, -1], dtype=torch.int32, device="cuda")
    if sizes is not None:
        off = offsets_of(sizes)
    bias = randn(g, n if sizes is None else (len(sizes), n), dt)
    want, size = grouped(xv, wv[None] if sizes is None else wv,
                         torch.tensor([0, m]) if off is None else off, rows=rows,
                         bias=bias[None] if sizes is None else bias, epi="elu")
    out = torch.full((many, n), 7.0, dtype=dt, device="cuda")

    def run():
        return tg.matmul_fp8(xq, wq, offsets=off, rows=rows, bias=bias, epilogue=tg.EPI_ELU,
                             out=out)

    got, names = kernels(run)
    ran(names, "fp8_kernel", want_shape)
    inside = ~torch.isnan(want[:, 0])
    own = 0.0 if dt == torch.float32 else 2.0 ** -12
    within(got[inside], want[inside], tolerance(want, size, k, dt, own)[inside], "y")
    assert bool((got[~inside] == 7).all())
    first = got.clone()
    for _ in range(3):   # equal calls, equal bits
        assert torch.equal(run(), first)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n,sizes,gather", [
    (2600, 1100, 4104, None, False),                       # nine blocks, none of them whole
    (2817, 1024, 4096, [1000, 0, 517, 1300], False),       # eight, the groups' ends ragged
    (700, 2000, 4000, [1, 1500, 0, 1100], True),           # rows twice, rows of zeros
])
def test_fp8_many_tiles(gpu, dtype, m, k, n, sizes, gather):
    """256 x 256 for 160 and more tiles of eight and more blocks and 16-bit
    results, 128 x 128 for fp32 ones."""
    check_fp8(DTYPES[dtype], m, k, n, sizes, gather, (128, 128) if dtype == "f32" else (256, 256))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n,sizes,gather", [
    (1500, 300, 200, [700, 0, 1, 799], False),
    (500, 900, 136, [3, 1200, 64, 0, 65, 700], True),
])
def test_fp8_small(gpu, dtype, m, k, n, sizes, gather):
    """64 x 64 for more than 1,024 tiles of 16 x 16 and fewer than 300 of 128 x
    128, in several groups."""
    check_fp8(DTYPES[dtype], m, k, n, sizes, gather, (64, 64))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n,sizes,gather", [
    (10_000, 400, 520, [5000, 0, 129, 4871], False),
    (3000, 130, 648, [1, 6000, 0, 3999], True),
])
def test_fp8_medium(gpu, dtype, m, k, n, sizes, gather):
    """128 x 128 for 300 and more tiles, of fewer than eight blocks."""
    check_fp8(DTYPES[dtype], m, k, n, sizes, gather, (128, 128))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,kb,n", [(1, 1, 16), (5, 3, 40), (33, 9, 130)])
def test_fp8_few_rows_keep_small_products(gpu, dtype, m, kb, n):
    """Large products that cancel leave the small ones beside them: each block
    sums to 240 * 240 - 240 * 240 + 126 / 8."""
    import tinygnn_amd as tg
    x, w = torch.full((m, kb, 128), 0.5), torch.full((n, kb, 128), 0.25)
    x[:, :, [3, 90]], w[:, :, 3], w[:, :, 90] = 240, 240, -240
    f8 = torch.float8_e4m3fn
    xq = tg.BlockRows(x.flatten(1).to("cuda", f8), torch.ones(kb, m, device="cuda"), kb * 128)
    wq = tg.BlockWeight(w.flatten(1).to("cuda", f8),
                        torch.ones(-(-n // 128), kb, device="cuda"), kb * 128)
    got, names = kernels(lambda: tg.matmul_fp8(xq, wq, dtype=DTYPES[dtype]))
    ran(names, "fp8_thin_kernel")
    assert torch.equal(got, torch.full((m, n), 15.75 * kb).to(DTYPES[dtype]).cuda())


def integers(g, shape, dt):
    """-1, 0 and 1: sums of up to 2^24 products are exact in fp32 in any order,
    so results equal the 64-bit sum rounded to their type."""
    return torch.randint(-1, 2, shape, generator=g, device="cuda").to(dt)


def gathered(g, m, x_rows):
    rows = torch.randint(0, x_rows, (m,), generator=g, device="cuda", dtype=torch.int32)
    rows[[0, m // 2]] = torch.tensor([x_rows, -1], dtype=torch.int32, device="cuda")
    return rows


HALF, FLOAT = ["bf16", "f16"], ["f32"]
RING = None


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtypes,sizes,k,n,shape,direct", [
    (HALF, [3, 0, 40, 1, 0], 72, 130, (32, 128), True),
    (HALF, [3, 0, 40, 1, 0], 71, 131, (32, 128), False),
    (HALF, [200, 0, 55], 64, 200, (64, 64), True),
    (HALF, [200, 0, 55], 65, 201, (64, 64), False),
    (HALF, [20000, 0, 1, 19999], 64, 130, (128, 128), True),
    (HALF, [20000, 0, 1, 19999], 33, 131, (128, 128), False),    # odd rows: by registers
    (HALF, [30000, 129, 9000], 257, 129, (128, 128), False),
    (HALF, [2000, 0, 3001], 1024, 2048, RING, True),
    (HALF, [2000, 0, 3001], 1160, 2056, RING, True),             # ends inside a part, a tile
    (FLOAT, [3, 0, 40, 1, 0], 71, 131, (32, 128), True),
    (FLOAT, [200, 0, 55], 65, 201, (64, 64), True),
    (FLOAT, [20000, 0, 1, 19999], 301, 100, (64, 128), True),
])
def test_grouped_forward(gpu, dtypes, sizes, k, n, shape, direct, gather, transpose):
    import tinygnn_amd as tg
    m, off = sum(sizes), offsets_of(sizes)
    for dt in (DTYPES[d] for d in dtypes):
        g = gen(m + k)
        x = integers(g, (m // 2 + 1 if gather else m, k), dt)
        rows = gathered(g, m, x.shape[0]) if gather else None
        w = integers(g, (len(sizes), n, k) if transpose else (len(sizes), k, n), dt)
        got, names = kernels(lambda: tg.grouped_matmul(x, w, off, rows=rows,
                                                       transpose=transpose))
        if shape is RING:
            ran(names, "grouped_ring_kernel")
        else:
            ran(names, "grouped_kernel", shape, [transpose, direct])
        want, _ = grouped(x, w, off, rows=rows, transpose=transpose)
        assert torch.equal(got, want.to(dt))


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtypes,sizes,k,n,shape,direct", [
    (HALF, [900, 0, 1, 355], 130, 200, (64, 64), True),
    (HALF, [900, 0, 1, 355], 131, 201, (64, 64), False),
    (HALF, [1537, 0, 1, 3462], 1030, 1032, (128, 128), True),     # parts of 512 rows
    (HALF, [1537, 0, 1, 3462], 1031, 1033, (128, 128), False),    # odd rows: by registers
    (HALF, [200 + 7 * (i % 23) for i in range(62)] + [5003, 0], 512, 2048, RING, True),
    (FLOAT, [900, 0, 1, 355], 131, 201, (64, 64), True),
    (FLOAT, [1537, 0, 1, 3462], 1031, 1033, (128, 128), True),
    (FLOAT + HALF, [0, 9000, 1, 40, 9001, 513], 70, 66, (64, 64), True),
    (FLOAT + HALF, [1_100_000, 3, 0, 700], 16, 16, (64, 64), True),
])
def test_grouped_gradient(gpu, dtypes, sizes, k, n, shape, direct, gather):
    """dw and dbias; the oracle without the last row of the largest group, or of
    one of its parts, differs."""
    import tinygnn_amd as tg
    m, off = sum(sizes), offsets_of(sizes)
    for dt in (DTYPES[d] for d in dtypes):
        g = gen(m + k)
        x = integers(g, (m // 2 + 1 if gather else m, k), dt)
        rows = gathered(g, m, x.shape[0]) if gather else None
        dy = integers(g, (m, n), dt)
        got, names = kernels(lambda: tg.grouped_matmul_wgrad(x, dy, off, rows=rows, bias=True))
        if shape is RING:
            ran(names, "wgrad_ring_kernel")
        else:
            ran(names, "wgrad_kernel", shape, [direct, True])
        dw, _, db, _ = wgrad(x, dy, off, rows=rows)
        assert torch.equal(got[0], dw.to(dt)) and torch.equal(got[1], db.to(dt))
        most = max(range(len(sizes)), key=lambda i: sizes[i])
        for p in (int(off[most + 1]) - 1, int(off[most]) + 511):
            r = p if rows is None else int(rows[p])
            row = x[r].double() if 0 <= r < x.shape[0] else x[0].double() * 0
            assert bool(row.any()) and bool(dy[p].any())
            less = dw[most] - row[:, None] * dy[p].double()[None]
            assert not torch.equal(got[0][most], less.to(dt))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_grouped_far_rows(gpu, dtype):
    """Rows gathered from places past 2^31 bytes: by registers, whatever the
    alignment."""
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(5)
    sizes, k, n = [20000, 0, 1, 22999, 300], 38, 100
    m, off = sum(sizes), offsets_of(sizes)
    lead = 2 ** 34 // torch.finfo(dt).bits // m + 200
    x = torch.empty(m, lead, dtype=dt, device="cuda")[:, :k]
    x.copy_(integers(g, (m, k), dt))
    rows = gathered(g, m, m)
    w, dy = integers(g, (len(sizes), k, n), dt), integers(g, (m, n), dt)
    got, names = kernels(lambda: tg.grouped_matmul(x, w, off, rows=rows))
    ran(names, "grouped_kernel", (64, 128 if dt == torch.float32 else 64), [False, False])
    assert torch.equal(got, grouped(x, w, off, rows=rows)[0].to(dt))
    got, names = kernels(lambda: tg.grouped_matmul_wgrad(x, dy, off, rows=rows, bias=True))
    ran(names, "wgrad_kernel", (64, 64), [False, True])
    dw, _, db, _ = wgrad(x, dy, off, rows=rows)
    assert torch.equal(got[0], dw.to(dt)) and torch.equal(got[1], db.to(dt))


def test_falling_offsets_of_many_rows(gpu):
    """Offsets that fall 512 times from m to 0 name 2^31 tiles and more of 64
    rows: rows of x and y alone are touched."""
    import tinygnn_amd as tg
    m, groups, guard = 3 << 27, 1024, 1 << 20
    off = torch.tensor([0, m] * 512 + [0], dtype=torch.int32, device="cuda")
    x = torch.full((m, 1), 2.0, device="cuda")
    out = torch.full((guard + m + guard, 1), 7.0, device="cuda")
    w = torch.full((groups, 1, 1), 3.0, device="cuda")
    tg.grouped_matmul(x, w, off, out=out[guard:guard + m])
    assert bool((out[:guard] == 7).all()) and bool((out[guard + m:] == 7).all())
    inside = out[guard:guard + m]
    assert bool(((inside == 6) | (inside == 7)).all()) and bool((inside == 6).any())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n", [(20, 300, 40), (1500, 300, 200), (10_000, 400, 520),
                                   (2600, 1100, 4104)])
@pytest.mark.parametrize("x_rows", [0, 50])
def test_fp8_rows_of_zeros_times_nan(gpu, dtype, m, k, n, x_rows):
    """An index outside x is a row of zeros in every tile shape, as in
    grouped_matmul: 0 times a NaN, in a weight or in a scale, is NaN."""
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(m)
    w = randn(g, (k, n), torch.float32)
    w[k // 2, 5] = float("nan")
    x = randn(g, (x_rows, k), torch.float32)
    rows = torch.full((m,), x_rows, dtype=torch.int32, device="cuda")
    if x_rows:
        rows[::2] = torch.randint(0, x_rows, (len(rows[::2]),), generator=g, device="cuda").int()
    got = tg.matmul_fp8(tg.quantize(x), tg.quantize_weight(w), rows=rows, dtype=dt)
    outside = rows == x_rows
    other = [i for i in range(n) if i != 5]
    assert torch.isnan(got[:, 5]).all() and not got[outside][:, other].any()
    assert torch.isfinite(got[:, other]).all()
    y = tg.grouped_matmul(x, w[None], offsets_of([m]), rows=rows)
    assert torch.equal(torch.isnan(y), torch.isnan(got))
