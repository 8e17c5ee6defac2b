"""Products grouped by expert or node type, and their e4m3 forms, on the GPU
against 64 bits.

Tolerances (u = 2^-24): a float32 sum of k products in any order is off by
(k + 2) u sum|a||b| at most (bias added: one more term), an ELU by 4 u more,
and the result is rounded to its type: half a step.  The e4m3 operands are
compared exactly (their definition's roundings are float32's), and the product
against those values: the sums within a block of 128, then of the blocks, with
two roundings of the scales.  Where the result has 16 bits, the e4m3 matrix
instructions' own sums come in: 2^-12 sum|a||b|."""
import pytest
import torch

from expert_cases import (DTYPES, U, e4m3, gen, grouped, half_step, least, offsets_of, padded,
                          randn, wgrad, within)

pytestmark = pytest.mark.gpu

EPILOGUES = ["none", "relu", "elu"]


def epi(tg, name):
    return dict(none=tg.EPI_NONE, relu=tg.EPI_RELU, elu=tg.EPI_ELU)[name]


def tolerance(want, size, k, dt):
    return ((k + 8) * U * size + half_step(dt) * (want.abs() + (k + 8) * U * size) + least(dt))


def tolerance_fp8(want, size, k, dt):
    own = 0.0 if dt == torch.float32 else 2.0 ** -12
    return tolerance(want, size, k, dt) + (1 + half_step(dt)) * own * size


def check_y(got, want, size, k, dt, tol=tolerance):
    inside = ~torch.isnan(want[:, 0]) if want.shape[1] else torch.zeros(0, dtype=torch.bool)
    within(got[inside], want[inside], tol(want, size, k, dt)[inside], "y")


SIZES = [[1], [0, 5, 0], [3, 0, 70, 1], [64, 64, 128], [17, 33, 200, 0, 1, 0], [300],
         [129, 255, 257]]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("k,n", [(1, 1), (5, 3), (16, 16), (64, 64), (32, 136), (129, 130),
                                 (200, 64), (602, 41), (256, 256), (96, 520), (1032, 72)])
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_grouped(gpu, sizes, k, n, dtype):
    """Forward with bias and epilogue, both layouts of w; the gradients."""
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(sum(sizes) + k * 3 + n)
    m, e = sum(sizes), len(sizes)
    off = offsets_of(sizes)
    x, dy = randn(g, (m, k), dt), randn(g, (m, n), dt)
    w, bias = randn(g, (e, k, n), dt, k ** -0.5), randn(g, (e, n), dt)
    name = EPILOGUES[(k + n) % 3]
    want, size = grouped(x, w, off, bias=bias, epi=name)
    check_y(tg.grouped_matmul(x, w, off, bias=bias, epilogue=epi(tg, name)), want, size, k, dt)
    wt = w.transpose(1, 2).contiguous()
    check_y(tg.grouped_matmul(x, wt, off, bias=bias, epilogue=epi(tg, name), transpose=True),
            want, size, k, dt)
    want, size = grouped(dy, w, off, transpose=True)
    check_y(tg.grouped_matmul(dy, w, off, transpose=True), want, size, n, dt)
    dw, dw_size, db, db_size = wgrad(x, dy, off)
    got_w, got_b = tg.grouped_matmul_wgrad(x, dy, off, bias=True)
    within(got_w, dw, tolerance(dw, dw_size, m, dt), "dw")
    within(got_b, db, tolerance(db, db_size, m, dt), "dbias")
    assert not got_w[[i for i, s in enumerate(sizes) if s == 0]].any()
    again = tg.grouped_matmul_wgrad(x, dy, off, bias=True)
    assert torch.equal(got_w, again[0]) and torch.equal(got_b, again[1])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("k,n,lead", [(64, 128, 0), (72, 40, 8), (33, 50, 1), (130, 66, 3)])
def test_grouped_rows_and_strides(gpu, dtype, k, n, lead):
    """Gathered rows (some of them outside x, some twice), leading dimensions,
    rows before and behind the groups left as they were."""
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(k + n)
    x = padded(randn(g, (90, k), dt), lead)
    rows = torch.randint(0, 90, (400,), generator=g, device="cuda", dtype=torch.int32)
    rows[[3, 77, 200]] = torch.tensor([-1, 90, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    off = torch.tensor([7, 7, 150, 151, 390], dtype=torch.int32, device="cuda")
    whole = randn(g, (4, k, n + lead), dt, k ** -0.5)
    w = whole[:, :, :n]
    want, size = grouped(x, w, off, rows=rows)
    out = padded(torch.full((400, n), 7.0, dtype=dt, device="cuda"), lead, 5.0)
    assert tg.grouped_matmul(x, w, off, rows=rows, out=out) is out
    check_y(out, want, size, k, dt)
    assert bool((out[:7] == 7).all()) and bool((out[390:] == 7).all())
    if lead:
        beyond = out.as_strided((400, lead), (n + lead, 1), out.storage_offset() + n)
        assert bool((beyond == 5).all())
    dy = padded(randn(g, (400, n), dt), lead)
    dw, dw_size, db, db_size = wgrad(x, dy, off, rows=rows)
    got_w, got_b = tg.grouped_matmul_wgrad(x, dy, off, rows=rows, bias=True)
    within(got_w, dw, tolerance(dw, dw_size, 400, dt), "dw")
    within(got_b, db, tolerance(db, db_size, 400, dt), "dbias")


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_grouped_nan_stays_in_its_group(gpu, dtype):
    """What lies outside a group's rows never reaches it: not NaN in other
    rows, nor in the columns behind a row, nor in other matrices."""
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(9)
    x = padded(randn(g, (200, 72), dt), 8)
    dy = padded(randn(g, (200, 80), dt), 8)
    w = randn(g, (3, 72, 80), dt)
    off = torch.tensor([10, 60, 61, 130], dtype=torch.int32, device="cuda")
    x[60:61] = float("nan")
    dy[60:61] = float("nan")
    x[130:], x[:10], dy[130:], dy[:10] = (float("nan"),) * 4
    w[1] = float("nan")
    y = tg.grouped_matmul(x, w, off)
    assert torch.isfinite(y[10:60]).all() and torch.isfinite(y[61:130]).all()
    assert torch.isnan(y[60]).all()
    dx = tg.grouped_matmul(dy, w, off, transpose=True)
    assert torch.isfinite(dx[10:60]).all() and torch.isfinite(dx[61:130]).all()
    dw, db = tg.grouped_matmul_wgrad(x, dy, off, bias=True)
    assert torch.isfinite(dw[[0, 2]]).all() and torch.isfinite(db[[0, 2]]).all()
    assert torch.isnan(dw[1]).all() and torch.isnan(db[1]).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_grouped_empty_sizes(gpu, dtype):
    import tinygnn_amd as tg
    dt = DTYPES[dtype]
    e = lambda *s: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
    off = offsets_of([0, 4])
    bias = torch.tensor([[1.0], [-2.0]], dtype=dt, device="cuda")
    y = tg.grouped_matmul(e(4, 0), e(2, 0, 1), off, bias=bias, epilogue=tg.EPI_RELU)
    assert y.flatten().tolist() == [0, 0, 0, 0]            # relu(-2)
    assert tg.grouped_matmul(e(4, 3), e(2, 3, 0), off).shape == (4, 0)
    assert tg.grouped_matmul(e(0, 3), e(2, 3, 5), offsets_of([0, 0])).shape == (0, 5)
    dw, db = tg.grouped_matmul_wgrad(e(0, 3), e(0, 5), offsets_of([0, 0]), bias=True)
    assert dw.shape == (2, 3, 5) and not dw.any() and not db.any()
    dw, db = tg.grouped_matmul_wgrad(e(4, 0), torch.ones(4, 5, dtype=dt, device="cuda"), off,
                                     bias=True)
    assert dw.shape == (2, 0, 5) and not db[0].any() and bool((db[1] == 4).all())


def test_grouped_many_rows_and_groups(gpu):
    """1,024 groups, most of them empty; more rows than 65,536 tiles of 16."""
    import tinygnn_amd as tg
    g = gen(11)
    sizes = [0] * 1024
    for i in range(0, 1024, 7):
        sizes[i] = i % 50
    sizes[1023] = 1_100_000
    off = offsets_of(sizes)
    m = sum(sizes)
    for dt in (torch.float32, torch.bfloat16):
        x, w = randn(g, (m, 16), dt), randn(g, (1024, 16, 16), dt)
        want, size = grouped(x, w, off)
        check_y(tg.grouped_matmul(x, w, off), want, size, 16, dt)
        dy = randn(g, (m, 16), dt)
        dw, dw_size, _, _ = wgrad(x, dy, off)
        got, _ = tg.grouped_matmul_wgrad(x, dy, off)
        # chains over the largest group's rows
        within(got, dw, tolerance(dw, dw_size, m, dt), "dw")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("k,n,gather", [(512, 2048, True), (520, 2056, False), (544, 1544, True),
                                        (602, 2048, False)])
def test_grouped_large_tiles(gpu, dtype, k, n, gather):
    """Sizes that take the 256-wide tiles and, with k or n of no whole chunks,
    those of 128: contractions that end inside a part, a group of more rows than
    their starts kept at once (2,048), empty groups, padded rows."""
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(k)
    sizes = [200 + 7 * (i % 23) for i in range(64)]
    sizes[3], sizes[5], sizes[40], sizes[63] = 5003, 0, 1, 0
    m, off = sum(sizes), offsets_of(sizes)
    x = padded(randn(g, (m // 2 if gather else m, k), dt), 8)
    rows = None
    if gather:
        rows = torch.randint(0, m // 2, (m,), generator=g, device="cuda", dtype=torch.int32)
        rows[[0, m // 3]] = torch.tensor([m // 2, -1], dtype=torch.int32, device="cuda")
    dy = padded(randn(g, (m, n), dt), 8)
    w, bias = randn(g, (64, k, n), dt, k ** -0.5), randn(g, (64, n), dt)
    want, size = grouped(x, w, off, rows=rows, bias=bias, epi="elu")
    y = tg.grouped_matmul(x, w, off, rows=rows, bias=bias, epilogue=tg.EPI_ELU)
    check_y(y, want, size, k, dt)
    want, size = grouped(dy, w, off, transpose=True)
    check_y(tg.grouped_matmul(dy, w, off, transpose=True), want, size, n, dt)
    dw, dw_size, db, db_size = wgrad(x, dy, off, rows=rows)
    got_w, got_b = tg.grouped_matmul_wgrad(x, dy, off, rows=rows, bias=True)
    # the longest chain is the largest group's
    within(got_w, dw, tolerance(dw, dw_size, 5003, dt), "dw")
    within(got_b, db, tolerance(db, db_size, 5003, dt), "dbias")
    again = tg.grouped_matmul_wgrad(x, dy, off, rows=rows, bias=True)
    assert torch.equal(got_w, again[0]) and torch.equal(got_b, again[1])


@pytest.mark.parametrize("groups", [None, 3])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_matmul_fp8_large_tiles(gpu, dtype, groups):
    import tinygnn_amd as tg
    dt, g, m, k, n = DTYPES[dtype], gen(17), 5003, 300, 8200
    xq, wq, xv, wv = fp8_operands(g, m, k, n, groups)
    off = None if groups is None else offsets_of([2000, 0, 3003])
    want, size = grouped(xv, wv[None] if groups is None else wv,
                         torch.tensor([0, m]) if off is None else off)
    got = tg.matmul_fp8(xq, wq, offsets=off, dtype=dt)
    check_y(got, want, size, k, dt, tolerance_fp8)


def test_grouped_bad_offsets_stay_inside(gpu):
    """Falling or outside offsets: only rows within x and y are touched."""
    import tinygnn_amd as tg
    x, w = torch.ones(50, 8, device="cuda"), torch.ones(3, 8, 8, device="cuda")
    off = torch.tensor([-5, 20, 10, 90], dtype=torch.int32, device="cuda")
    out = torch.zeros(60, 8, device="cuda")
    tg.grouped_matmul(x, w, off, out=out[:50])
    assert bool((out[:50] == 8).all()) and not out[50:].any()
    dw, _ = tg.grouped_matmul_wgrad(x, x, off)
    assert bool((dw[0] == 20).all()) and not dw[1].any() and bool((dw[2] == 40).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 127), (64, 128), (33, 129), (7, 1000), (3, 4096),
                                       (2708, 1433)])
def test_quantize(gpu, rows, cols, dtype):
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(rows + cols)
    x = padded(randn(g, (rows, cols), dt, 10.0), 3)
    x[0, :: 3] = 0
    if rows > 4:
        x[1], x[2], x[3] = 0, torch.finfo(dt).max, torch.finfo(dt).smallest_normal
    _, q, scale = e4m3(x)
    got = tg.quantize(x)
    assert got.q.shape == q.shape and got.scale.shape == scale.t().shape
    assert torch.equal(got.scale, scale.t())
    assert torch.equal(got.q.view(torch.uint8) & 0x7F, q.view(torch.uint8) & 0x7F)
    assert torch.equal(got.q.float(), q.float())


def test_quantize_bad_values(gpu):
    """A NaN stays one NaN, an infinity makes its block NaN, others stay."""
    import tinygnn_amd as tg
    x = torch.ones(3, 256, device="cuda")
    x[0, 5], x[1, 200] = float("nan"), float("inf")
    got = tg.quantize(x)
    value = got.q.float() * got.scale.t().repeat_interleave(128, 1)
    assert torch.isnan(value[0, 5]) and int(torch.isnan(value[0]).sum()) == 1
    assert torch.isfinite(value[1, :128]).all() and torch.isnan(value[1, 128:]).all()
    assert torch.isfinite(value[2]).all()


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("k,n", [(1, 1), (128, 128), (200, 130), (64, 300), (1433, 16)])
def test_quantize_weight(gpu, k, n, transpose):
    import tinygnn_amd as tg
    w = randn(gen(k + n), (2, k, n), torch.bfloat16)
    got = tg.quantize_weight(w.transpose(1, 2).contiguous() if transpose else w, transpose)
    nb, kb = -(-n // 128), -(-k // 128)
    full = torch.zeros(2, nb * 128, kb * 128, device="cuda")
    full[:, :n, :k] = w.transpose(1, 2).float()
    blocks = full.view(2, nb, 128, kb, 128)
    scale = (blocks.abs().amax((2, 4)) * (1 / 448)).clamp_min(2.0 ** -126)
    q = (blocks / scale[:, :, None, :, None]).to(torch.float8_e4m3fn).view(2, nb * 128, kb * 128)
    assert got.k == k and torch.equal(got.scale, scale)
    assert torch.equal(got.q.float(), q[:, :n].float())
    one = tg.quantize_weight(w[1])
    assert torch.equal(one.q.float(), got.q[1].float()) and torch.equal(one.scale, got.scale[1])


def fp8_operands(g, m, k, n, e=None, dt=torch.bfloat16):
    """Quantised operands and their values in 64 bits."""
    import tinygnn_amd as tg
    lead = () if e is None else (e,)
    x, w = randn(g, (m, k), dt), randn(g, (*lead, k, n), dt, k ** -0.5)
    xq, wq = tg.quantize(x), tg.quantize_weight(w)
    wide = wq.scale.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)
    wv = (wq.q.double() * wide)[..., :k].transpose(-1, -2)
    return xq, wq, e4m3(x)[0], wv


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (5, 128, 16), (3, 200, 130), (16, 1024, 64),
                                   (17, 4096, 48), (128, 256, 128), (300, 384, 257),
                                   (257, 129, 520), (1000, 640, 384)])
def test_matmul_fp8(gpu, m, k, n, dtype):
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(m + k + n)
    xq, wq, xv, wv = fp8_operands(g, m, k, n)
    bias = randn(g, n, dt)
    name = EPILOGUES[m % 3]
    want, size = grouped(xv, wv[None], torch.tensor([0, m]), bias=bias[None], epi=name)
    got = tg.matmul_fp8(xq, wq, bias=bias, epilogue=epi(tg, name), dtype=dt)
    within(got, want, tolerance_fp8(want, size, k, dt), "y")


@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("k,n", [(128, 128), (300, 200)])
def test_matmul_fp8_groups(gpu, sizes, k, n):
    import tinygnn_amd as tg
    g, e, dt = gen(sum(sizes) + k), len(sizes), torch.bfloat16
    xq, wq, xv, wv = fp8_operands(g, 90, k, n, e)
    m = sum(sizes) + 9
    rows = torch.randint(0, 90, (m,), generator=g, device="cuda", dtype=torch.int32)
    rows[m // 2] = 90                                      # outside: a row of zeros
    off = offsets_of(sizes) + 4
    bias = randn(g, (e, n), dt)
    want, size = grouped(xv, wv, off, rows=rows, bias=bias)
    out = torch.full((m, n), 7.0, dtype=dt, device="cuda")
    tg.matmul_fp8(xq, wq, offsets=off, rows=rows, bias=bias, out=out)
    check_y(out, want, size, k, dt, tolerance_fp8)
    assert bool((out[:4] == 7).all()) and bool((out[4 + sum(sizes):] == 7).all())


def test_matmul_fp8_empty(gpu):
    import tinygnn_amd as tg
    x, w = torch.empty(0, 40, device="cuda"), torch.ones(40, 7, device="cuda")
    assert tg.matmul_fp8(tg.quantize(x), tg.quantize_weight(w)).shape == (0, 7)
    x, w = torch.empty(3, 0, device="cuda"), torch.empty(0, 7, device="cuda")
    y = tg.matmul_fp8(tg.quantize(x), tg.quantize_weight(w), bias=torch.ones(7, device="cuda"))
    assert bool((y == 1).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_grouped_wgrad_whole_and_cut_groups(gpu, dtype):
    """Groups of no row, of few and of many: some are cut to parts of rows,
    some are one part; each group's tolerance counts its own rows."""
    import tinygnn_amd as tg
    dt = DTYPES[dtype]
    sizes = [9000, 0, 1, 40, 9001, 513, 0]
    off = offsets_of(sizes)
    g = gen(11)
    x, dy = randn(g, (sum(sizes), 70), dt), randn(g, (sum(sizes), 66), dt)
    dw, db = tg.grouped_matmul_wgrad(x, dy, off, bias=True)
    assert tg.lib.tg_grouped_matmul_wgrad_workspace_size(sum(sizes), 70, 66, len(sizes),
                                                         tg.TYPE_F32) > 0
    want_w, size_w, want_b, size_b = wgrad(x, dy, off)
    n = torch.tensor(sizes, device="cuda").double()
    within(dw, want_w, tolerance(want_w, size_w, n[:, None, None], dt), "dw")
    within(db, want_b, tolerance(want_b, size_b, n[:, None], dt), "dbias")


def test_grouped_wgrad_bias_only(gpu):
    """The C entry with dw NULL, in a workspace of the size asked for."""
    import tinygnn_amd as tg
    m, k, n, groups = 40000, 1024, 512, 64
    off = torch.linspace(0, m, groups + 1, device="cuda").int()
    dy = randn(gen(3), (m, n), torch.float32)
    size = tg.lib.tg_grouped_matmul_wgrad_workspace_size(m, k, n, groups, tg.TYPE_F32)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    db = torch.empty(groups, n, device="cuda")
    tg.lib.check(tg.lib.tg_grouped_matmul_wgrad(
        m, k, n, groups, tg.TYPE_F32, None, m, k, None, dy.data_ptr(), n, off.data_ptr(), None,
        db.data_ptr(), ws.data_ptr(), size, tg.stream_handle()))
    _, _, want, bound = wgrad(dy[:, :1], dy, off)
    within(db, want, tolerance(want, bound, m // groups, torch.float32), "dbias")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("far", [False, True])
def test_grouped_many_wide_tiles(gpu, dtype, far):
    """Tiles enough for the wider shapes; far: gathered from rows whose places
    pass 2^31 bytes."""
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(5)
    sizes, k, n = [20000, 0, 1, 22999, 300], 38, 100
    m, off = sum(sizes), offsets_of(sizes)
    lead = 2 ** 34 // torch.finfo(dt).bits // m + 200 if far else 40
    x = torch.empty(m, lead, dtype=dt, device="cuda")[:, :k]
    x.copy_(randn(g, (m, k), dt))
    rows = torch.randperm(m, generator=g, device="cuda").int()
    rows[5], rows[-1] = -1, m
    w, bias = randn(g, (len(sizes), k, n), dt, k ** -0.5), randn(g, (len(sizes), n), dt)
    want, size = grouped(x, w, off, rows=rows, bias=bias, epi="elu")
    got = tg.grouped_matmul(x, w, off, rows=rows, bias=bias, epilogue=tg.EPI_ELU)
    check_y(got, want, size, k, dt)
    wt = w.transpose(1, 2).contiguous()
    got = tg.grouped_matmul(x, wt, off, rows=rows, bias=bias, epilogue=tg.EPI_ELU, transpose=True)
    check_y(got, want, size, k, dt)
    dy = randn(g, (m, n), dt)
    dw, dw_size, db, db_size = wgrad(x, dy, off, rows=rows)
    got, got_b = tg.grouped_matmul_wgrad(x, dy, off, rows=rows, bias=True)
    count = torch.tensor(sizes, device="cuda").double()
    within(got, dw, tolerance(dw, dw_size, count[:, None, None], dt), "dw")
    within(got_b, db, tolerance(db, db_size, count[:, None], dt), "dbias")


@pytest.mark.parametrize("count,k", [(2 ** 24 + 77, 128), (2 ** 22 + 77, 600)])
def test_matmul_fp8_far_rows(gpu, count, k):
    """Rows gathered from places past 2^31 bytes: the same values as from a
    copy of those rows, whose products run in the same order."""
    import tinygnn_amd as tg
    g, n, m = gen(9), 40, 20000
    x = torch.zeros(count, k, dtype=torch.bfloat16, device="cuda")
    rows = torch.randint(0, count, (m,), generator=g, device="cuda").int()
    rows[0], rows[1] = count - 1, 0
    x[rows.long()] = randn(g, (m, k), torch.bfloat16)
    xq, wq = tg.quantize(x), tg.quantize_weight(randn(g, (k, n), torch.bfloat16))
    del x
    near = tg.BlockRows(xq.q[rows.long()].contiguous(), xq.scale[:, rows.long()].contiguous(), k)
    v = near.q.double() * near.scale.double().t().repeat_interleave(128, 1)
    wv = wq.q.double() * wq.scale.double().repeat_interleave(128, 1)
    want, size = v @ wv.t(), v.abs() @ wv.abs().t()
    rows[2] = count
    want[2] = size[2] = 0
    for dt in (torch.float32, torch.bfloat16):
        got = tg.matmul_fp8(xq, wq, rows=rows, dtype=dt)
        within(got, want, tolerance_fp8(want, size, k, dt), "y")
        same = tg.matmul_fp8(near, wq, dtype=dt)
        same[2] = 0
        assert torch.equal(got, same)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n", [(3, 6, 5), (300, 512, 264)])
def test_gathered_from_no_rows(gpu, dtype, m, k, n):
    """Every index is outside an x of no rows: rows of zeros, plus the bias."""
    import tinygnn_amd as tg
    dt, off = DTYPES[dtype], offsets_of([m - 1, 1])
    x = torch.empty(0, k, dtype=dt, device="cuda")
    rows = torch.arange(-1, m - 1, dtype=torch.int32, device="cuda")
    bias = torch.stack([torch.ones(n), torch.full((n,), 2.0)]).to(dt).cuda()
    want = torch.cat([bias[:1].expand(m - 1, n), bias[1:]])
    for t in (False, True):
        w = torch.ones(2, *((n, k) if t else (k, n)), dtype=dt, device="cuda")
        assert torch.equal(tg.grouped_matmul(x, w, off, rows=rows, bias=bias, transpose=t), want)
    wq = tg.quantize_weight(w, transpose=True)
    got = tg.matmul_fp8(tg.quantize(x), wq, offsets=off, rows=rows, bias=bias, dtype=dt)
    assert torch.equal(got, want)
    dw, db = tg.grouped_matmul_wgrad(x, torch.ones(m, n, dtype=dt, device="cuda"), off, rows=rows,
                                     bias=True)
    assert not dw.any() and torch.equal(db[:, 0], torch.tensor([m - 1, 1], device="cuda").to(dt))
