"""The workspace of the weights' gradient: sums of the parts of groups that are
cut, and of no others."""
import pytest
import torch

from expert_cases import gen, offsets_of, wgrad


def size(m, k, n, groups, kind=0):
    import tinygnn_amd as tg
    return tg.lib.tg_grouped_matmul_wgrad_workspace_size(m, k, n, groups, kind)


@pytest.mark.parametrize("m,k,n,groups,cut", [
    (20_000, 4096, 4096, 64, 1),      # parts of 16,384 rows: one group can be cut, in two
    (60_000, 1024, 2048, 500, 3),
    (16_384, 4096, 4096, 64, 0),
])
def test_size_follows_what_can_be_cut(m, k, n, groups, cut):
    """`cut` groups in `cut` more parts than groups at most."""
    assert size(m, k, n, groups) <= 2 * cut * (k + 1) * n * 4 + 512
    assert (size(m, k, n, groups) > 0) == (cut > 0)


def integers(g, shape):
    return torch.randint(-1, 2, shape, generator=g, device="cuda").float()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,k,n", [
    ([16384, 16385, 0, 1, 32768, 32769, 5, 100], 1024, 1024),   # whole parts and one row more
    ([0, 16384 * 3 + 1], 2048, 2048),
    ([512, 513, 0, 1024, 1025, 7, 4096, 0, 1], 33, 40),         # parts of 512
    ([700, 511, 1537], 130, 70),
])
@pytest.mark.parametrize("kind", [0, 1])
def test_cut_groups(gpu, sizes, k, n, kind):
    """Sums of whole numbers are exact: equal to 64 bits rounded once.  Nothing
    is written behind the workspace."""
    import tinygnn_amd as tg
    dt = {0: torch.float32, 1: torch.bfloat16}[kind]
    g, m, off = gen(m_ := sum(sizes)), m_, offsets_of(sizes)
    x, dy = integers(g, (m, k)).to(dt), integers(g, (m, n)).to(dt)
    need = size(m, k, n, len(sizes), kind)
    ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    dw = torch.full((len(sizes), k, n), 9.0, dtype=dt, device="cuda")
    db = torch.full((len(sizes), n), 9.0, dtype=dt, device="cuda")

    def run(offsets):
        tg.lib.check(tg.lib.tg_grouped_matmul_wgrad(
            m, k, n, len(sizes), kind, x.data_ptr(), m, k, None, dy.data_ptr(), n,
            offsets.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), need,
            tg.stream_handle()))
        assert bool((ws[need:] == 0x5A).all())

    want, _, want_b, _ = wgrad(x, dy, off)
    run(off)
    assert torch.equal(dw, want.to(dt)) and torch.equal(db, want_b.to(dt))
    # one row left out of a cut group shows
    at = max(range(len(sizes)), key=lambda i: sizes[i])
    row = int(off[at]) + sizes[at] // 2
    less = want[at] - x[row].double()[:, None] * dy[row].double()[None]
    assert not torch.equal(dw[at], less.to(dt))
    # falling offsets name more parts than there are: nothing outside is touched
    wild = torch.tensor([0, m] * len(sizes), dtype=torch.int32, device="cuda")[:len(sizes) + 1]
    run(wild.contiguous())
