"""Each tile shape of the grouped and e4m3 products, by the kernel that ran,
at sizes from both sides of the rules that choose it, against 64 bits.

Tolerances (u = 2^-24) as in test_grouped_gpu: a float32 sum of k products is
off by (k + 8) u sum|a||b| at most, bias and epilogue among it, the result
rounded to its type; e4m3 products of 16-bit results by 2^-12 sum|a||b| more."""
import re

import pytest
import torch

from expert_cases import DTYPES, U, e4m3, gen, grouped, half_step, least, offsets_of, randn, within

pytestmark = pytest.mark.gpu


def kernels(fn):
    """fn's result and the names of the kernels that it ran."""
    from torch.profiler import ProfilerActivity, profile
    with profile(activities=[ProfilerActivity.CUDA], acc_events=True) as p:
        out = fn()
        torch.cuda.synchronize()
    return out, [e.key for e in p.key_averages()]


def shape_of(names, kernel):
    """(rows, columns) of the tile of the one kernel of a name, which is mangled
    or not, as the profiler can."""
    found = [n for n in names if re.search(rf"(\b|\d){kernel}(<|I)", n)]
    assert len(found) == 1, (kernel, names)
    shape = re.search(r"Shape(?:<|ILi)(\d+)(?:, |ELi)(\d+)", found[0])
    return int(shape[1]), int(shape[2])


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
    assert shape_of(names, "fp8_kernel") == want_shape
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
