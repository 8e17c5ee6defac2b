"""Each tile of the dense layers' products in its three layouts (x w, x w^T, x^T dy),
whole and cut along the contraction, with operands straight to LDS, through
registers and through the large tile's ring: by the kernel that ran.  Operands are
-1, 0 and 1, so that sums are exact and one value lost or taken twice shows."""
import pytest
import torch

from expert_cases import DTYPES, gen, padded
from test_linear_sums_gpu import exact, integers
from test_tile_shapes_gpu import kernels, ran

pytestmark = pytest.mark.gpu
HALF, FLOAT = ["bf16", "f16"], ["f32"]
FEW, SMALL, WIDE, TALL, MEDIUM = (32, 128), (64, 64), (64, 128), (128, 64), (128, 128)
RING = None
LAYOUTS = {"y": [False, True], "transposed": [False, False], "dw": [True, True]}


def product(x, w, layout):
    """out = x @ w, x [m, k] and w [k, n], by the layout's call, with the bias -1 and
    ReLU where it has one: (out, the kernels that ran)."""
    import tinygnn_amd as tg
    m, n = x.shape[0], w.shape[1]
    if layout == "dw":
        x = far_of(x, x.t())
        dw = torch.empty(m, n, dtype=x.dtype, device="cuda")
        kind = tg._Torch().types[x.dtype]
        size = tg.lib.tg_linear_workspace_size(m, len(x), n, kind) + 256
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")

        def call():
            tg.lib.check(tg.lib.tg_linear_backward(
                len(x), m, n, kind, w.data_ptr(), w.stride(0), x.data_ptr(), x.stride(0), None, n,
                0, None, 0, 0, None, 0, dw.data_ptr(), None, ws.data_ptr(), size,
                tg.stream_handle()))
            return dw
        return kernels(call)
    x = far_of(x, x)
    bias = torch.full((n,), -1.0, dtype=x.dtype, device="cuda")
    w = w.t().contiguous() if layout == "transposed" else w
    return kernels(lambda: tg.linear(x, w, bias=bias, epilogue=tg.EPI_RELU,
                                     transpose=layout == "transposed"))


def far_of(x, t):
    """t's values, in rows as far apart as x.far says."""
    lead = getattr(x, "far", 0)
    return padded(t, lead, fill=0.0) if lead else t.contiguous()


def check(m, k, n, dt, layout, shape, direct, far=0):
    g = gen(m + 3 * k + n)
    x, w = integers(g, (m, k), dt), integers(g, (k, n), dt)
    x.far = far
    want = exact(x, w)
    if layout != "dw":
        want = (want - 1).clamp_min(0)
    got, names = product(x, w, layout)
    if shape is RING:
        ran(names, "linear_ring_kernel")
    else:
        ran(names, "linear_kernel", shape, LAYOUTS[layout] + [direct])
    assert torch.equal(got, want.to(dt))
    for _ in range(2):   # equal calls, equal bits
        assert torch.equal(product(x, w, layout)[0], got)


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("dtypes,m,k,n,shape,direct", [
    # 16 bits, odd rows: through registers
    (HALF, 131, 301, 67, SMALL, False),
    (HALF, 301, 71, 131, SMALL, False),
    (HALF, 17, 20_001, 131, SMALL, False),
    (HALF, 2901, 71, 4101, MEDIUM, False),
    (HALF, 1101, 1101, 16_401, MEDIUM, False),
    (HALF, 1101, 5001, 1501, MEDIUM, False),
    (HALF, 2805, 28_511, 1973, MEDIUM, False),
    (HALF, 1973, 9001, 2805, MEDIUM, False),
    # rows of whole dwords: straight to LDS
    (HALF, 22, 1102, 2902, FEW, True),
    (HALF, 22, 70, 16_402, FEW, True),
    (HALF, 130, 1102, 22, SMALL, True),
    (HALF, 302, 70, 130, SMALL, True),
    (HALF, 702, 5002, 1102, WIDE, True),
    (HALF, 1502, 302, 2102, WIDE, True),
    (HALF, 2102, 5002, 130, TALL, True),
    (HALF, 16_402, 302, 130, TALL, True),
    (HALF, 702, 20_002, 1102, MEDIUM, True),
    (HALF, 2902, 70, 4102, MEDIUM, True),
    # whole chunks: the large tile
    (HALF, 1504, 20_000, 136, RING, True),
    (HALF, 6000, 5000, 136, RING, True),
    (HALF, 2904, 72, 4104, RING, True),
    (FLOAT, 21, 301, 4101, FEW, True),
    (FLOAT, 21, 71, 16_401, FEW, True),
    (FLOAT, 21, 301, 23, SMALL, True),
    (FLOAT, 133, 71, 23, SMALL, True),
    (FLOAT, 301, 20_001, 1501, WIDE, True),
    (FLOAT, 1501, 71, 2101, WIDE, True),
    (FLOAT, 1101, 5001, 21, TALL, True),
    (FLOAT, 16_401, 71, 131, TALL, True),
])
def test_tiles(gpu, dtypes, m, k, n, shape, direct, layout):
    for d in dtypes:
        check(m, k, n, DTYPES[d], layout, shape, direct)


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n", [(130, 300, 68), (300, 40, 131), (33, 700, 24)])
def test_rows_past_two_gigabytes(gpu, dtype, m, k, n, layout):
    """256 rows that reach past 2 GB: through registers, fp32 as well."""
    dt = DTYPES[dtype]
    check(m, k, n, dt, layout, SMALL, False, far=2 ** 31 // 256 // dt.itemsize)


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,n", [(128, 40_000, 24), (32, 40_000, 16), (24, 233_001, 41),
                                   (70, 6000, 8), (602, 30_011, 256)])
def test_exact_long_contractions(gpu, dtype, m, k, n, layout):
    """As many parts as a contraction is cut in."""
    dt, g = DTYPES[dtype], gen(k)
    x, w = integers(g, (m, k), dt), integers(g, (k, n), dt)
    want = exact(x, w)
    if layout != "dw":
        want = (want - 1).clamp_min(0)
    assert torch.equal(product(x, w, layout)[0], want.to(dt))
