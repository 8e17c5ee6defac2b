"""Long contractions of the dense layers and their gradients: sums of one sign, and
sums that are exact, where one value lost or taken twice shows."""
import pytest
import torch

import head_cases as hc
from expert_cases import DTYPES, gen, half_step, within

pytestmark = pytest.mark.gpu
U = hc.U


@pytest.mark.parametrize("layout", ["dw", "y", "transposed"])
@pytest.mark.parametrize("dtype,k", [("f16", 262_144), ("bf16", 2_097_152)])
def test_one_sign_of_16_bits(gpu, dtype, k, layout):
    """4,096 x 4,096 tiles fill the card without a cut.  The sums of equal values round
    the same way each time: a chain of n such values, added eight at a time by half a
    step of 2^-24, is off by n 2^-27 of its sum at most, and chains stop at 32,768
    values (bf16 262,144), half of the result's rounding; their sums are a chain of 64
    at most."""
    import tinygnn_amd as tg
    dt, n = DTYPES[dtype], 4096
    g = gen(k)
    a, c = (1 + torch.rand(2, n, generator=g, device="cuda")).to(dt)
    c = c / 32
    want = k * a.double()[:, None] * c.double()
    if layout == "dw":
        got = tg.linear_backward(c.expand(k, n).contiguous(), a.expand(k, n).contiguous(),
                                 torch.ones(n, n, dtype=dt, device="cuda"))[1]
    else:
        rows = c[:, None].expand(n, k) if layout == "transposed" else c.expand(k, n)
        got = tg.linear(a[:, None].expand(n, k).contiguous(), rows.contiguous(),
                        transpose=layout == "transposed")
    own = (half_step(dt) / 2 + 66 * U) * want
    within(got, want, own + half_step(dt) * (want + own), layout)
