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


def integers(g, shape, dt):
    """-1, 0 and 1: sums of up to 2^24 products are exact in float32 in any order."""
    return torch.randint(-1, 2, shape, generator=g, device="cuda").to(dt)


def exact(x, w):
    """x @ w of integers: sums of 4,096 products, exact in float32, in 64 bits."""
    out = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    for at in range(0, x.shape[1], 4096):
        out += x[:, at:at + 4096].float() @ w[at:at + 4096].float()
    return out


@pytest.mark.parametrize("layout", ["dw", "y", "transposed"])
@pytest.mark.parametrize("dtype,m,k,n", [
    ("f32", 8192, 100_001, 8000),    # 7 parts, 4 at a time
    ("f16", 8192, 200_004, 8000),    # in whole chunks: 7 parts of the large tile
    ("f16", 8191, 200_001, 8001),    # through registers
    ("f32", 12_000, 40_000, 12_004),  # 3 parts, 2 at a time
    ("f32", 2056, 300_000, 1032),    # 19 parts at once
])
def test_parts_at_a_time(gpu, dtype, m, k, n, layout):
    import tinygnn_amd as tg
    dt, g = DTYPES[dtype], gen(m)
    x, w = integers(g, (m, k), dt), integers(g, (k, n), dt)
    want = exact(x, w)
    if layout == "dw":
        x = x.t().contiguous()
        got = tg.linear_backward(w, x, torch.ones(m, n, dtype=dt, device="cuda"))[1]
    else:
        bias, residual = integers(g, (n,), dt), integers(g, (m, n), dt)
        if layout == "transposed":
            w = w.t().contiguous()
        got, pre = tg.linear(x, w, bias=bias, residual=residual, epilogue=tg.EPI_RELU,
                             transpose=layout == "transposed", with_pre=True)
        want += bias
        assert torch.equal(pre, want.to(dt))
        want = want.clamp_min(0) + residual
    assert torch.equal(got, want.to(dt))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_memory_of_a_plain_backward(gpu, dtype):
    """A product without an epilogue: dx, dw and dbias with its few parts, no d."""
    import tinygnn_amd as tg
    dt = DTYPES[dtype]
    m, k, n = 16_384, 1024, 8192
    x, w, dy = (torch.zeros(s, dtype=dt, device="cuda") for s in ((m, k), (k, n), (m, n)))
    for _ in range(2):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = tg.linear_backward(dy, x, w, bias=True)
        used = torch.cuda.max_memory_allocated() - before
        parts = tg.lib.tg_linear_workspace_size(k, m, n, tg.TYPE_F32 if dt == torch.float32 else
                                                tg.TYPE_BF16)
        results = sum(t.numel() * t.element_size() for t in out)
        assert used <= results + parts + 16 * 2 ** 20, (used, results, parts)
        del out


@pytest.mark.parametrize("m,k,n", [(1, 300_000, 41), (512, 300_001, 520), (2056, 300_001, 1032),
                                   (128, 40_000, 24)])
def test_one_sign_of_floats(gpu, m, k, n):
    """Chains of 256 values, 64 of those at most in a part, 512 parts at most in a
    chain of their own: that many steps of 2^-24, of sums that only grow."""
    import tinygnn_amd as tg
    g = gen(k)
    x, dy = (1 + torch.rand((k, c), generator=g, device="cuda") for c in (m, n))
    want = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for at in range(0, k, 50_000):
        want += x[at:at + 50_000].double().t().contiguous() @ dy[at:at + 50_000].double()
    parts = tg.lib.tg_linear_workspace_size(m, k, n, tg.TYPE_F32) // (4 * m * n)
    assert 0 < parts <= 512
    for got in (tg.linear_backward(dy, x, torch.ones(m, n, device="cuda"))[1],
                tg.linear(x.t().contiguous(), dy),
                tg.linear(x.t().contiguous(), dy.t().contiguous(), transpose=True)):
        within(got, want, (256 + 64 + parts + 2) * U * want, "sums")


def test_parts_at_a_time_captured(gpu):
    """The launches of later parts in a graph: replayed on new inputs, eager calls with a
    workspace of their own in between."""
    import tinygnn_amd as tg
    g, m, k, n = gen(9), 12_000, 40_000, 12_004
    x, w = integers(g, (m, k), torch.float32), integers(g, (k, n), torch.float32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tg.linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = tg.linear(x, w)
    for _ in range(3):
        x.copy_(integers(g, (m, k), torch.float32))
        want = tg.linear(x, w)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    assert torch.equal(y, exact(x, w).float())
