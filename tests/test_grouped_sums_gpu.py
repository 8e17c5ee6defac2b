"""fp32 sums of the grouped products keep their digits, whatever their length.

A sum of n values runs in chains of 256 that are added up, parts of 16,384 rows
in the weights' gradient: off by (256 + n / 256 + parts + 2) u of a sum of
positive values at most, u = 2^-24.  The values are 1 and v = 1 + (1 - 2^-10) h:
where one chain has passed 1 / u times 2 h (half a step of it is h), every
addition of v loses all but 1."""
import pytest
import torch

from expert_cases import U, offsets_of

pytestmark = pytest.mark.gpu


def loses(half):
    return 1 + half * (1 - 2 ** -10)


@pytest.mark.parametrize("m,n,groups", [(3, 130, 1), (300, 64, 2), (20000, 130, 2),
                                        (40000, 128, 1)])
@pytest.mark.parametrize("transpose", [False, True])
def test_products(gpu, m, n, groups, transpose):
    """k = 8,191: from 4,096 on a step is 2^-11.  One chain is off by 2,048 u."""
    import tinygnn_amd as tg
    k, v = 8191, loses(2.0 ** -12)
    x = torch.ones(m, k, device="cuda")
    w = torch.full((groups, n, k) if transpose else (groups, k, n), v, device="cuda")
    off = offsets_of([m // groups] * groups)
    y = tg.grouped_matmul(x, w, off, transpose=transpose)
    assert float((y.double() - k * v).abs().max()) <= (256 + k / 256 + 2) * U * k * v


@pytest.mark.parametrize("m,k,n,groups", [
    (100_000, 2048, 2048, 1),    # parts of m / 4 rows by the number of tiles alone
    (30_000, 2048, 2048, 2),     # tiles enough for whole groups
    (16_000, 1600, 2048, 1),
    (200_000, 70, 40, 2),        # many short parts
])
def test_gradient_of_weights(gpu, m, k, n, groups):
    """Chains of 16,384 rows and more: a step is 2^-9 from 2^14 on, and below it
    the values round up.  One chain of 25,000 is off by 5,600 u."""
    import tinygnn_amd as tg
    v = loses(2.0 ** -10 if m // groups > 20_000 else 2.0 ** -11)
    x = torch.ones(m, k, device="cuda")
    dy = torch.full((m, n), v, device="cuda")
    dw, db = tg.grouped_matmul_wgrad(x, dy, offsets_of([m // groups] * groups), bias=True)
    rows = m // groups
    parts = 2 + rows // 512
    tol = (256 + min(rows, 16384) / 256 + parts + 2) * U * rows * v
    assert float((dw.double() - rows * v).abs().max()) <= tol
    assert float((db.double() - rows * v).abs().max()) <= tol


def test_bias_beside_large_tiles(gpu):
    """dbias of 2^20 rows in fp16, 65,536 to each of 16 wavefronts: a chain of
    them from 2^14 on drops 2^-10 of every v = 1 + 2^-10, 7e-4 in all, where the
    result's own rounding is 4.9e-4."""
    import tinygnn_amd as tg
    m, k, n = 1 << 20, 4096, 8192
    v = (1 + 2.0 ** -10) / 256      # the sum is 4,100
    x = torch.ones(m, k, dtype=torch.float16, device="cuda")
    dy = torch.full((m, n), v, dtype=torch.float16, device="cuda")
    _, db = tg.grouped_matmul_wgrad(x, dy, offsets_of([m]), bias=True)
    assert bool((db == 4100).all())
