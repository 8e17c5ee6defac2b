"""What the size functions of the dense layers ask for, without a GPU."""
import pytest

from tinygnn_amd import _lib

F32, BF16, F16 = 0, 1, 2
GB = 1 << 30


@pytest.mark.parametrize("m,k,n,kind", [
    (8192, 1_000_000, 8192, F32), (8192, 10_000_000, 8192, F16), (8192, 20_000_000, 8192, BF16),
    (602, 100_000_000, 256, F32), (1, 2 ** 31 - 5000, 4096, F32), (32, 2 ** 31 - 5000, 4096, F16),
])
def test_parts_of_long_contractions(m, k, n, kind):
    """Sums of at most 1 GB stand at a time, however many parts there are."""
    L = _lib.lib.load()
    for need in (L.tg_linear_workspace_size(m, k, n, kind),
                 L.tg_linear_backward_workspace_size(k, m, n, kind) - _beside(k, n, kind)):
        assert 0 < need <= GB


def _beside(m, n, kind):
    """Bytes of d, and of dbias' parts at the most (1,024 of them and a part of columns)."""
    return m * n * (4 if kind == F32 else 2) + 4 * 1024 * (n + 512)


@pytest.mark.parametrize("kind", [F32, F16])
def test_parts_of_large_results(kind):
    """Two at the least: the sum of those before, and the next."""
    L = _lib.lib.load()
    m = n = 40_000
    assert L.tg_linear_workspace_size(m, 1_000_000, n, kind) == 2 * 4 * m * n
    assert L.tg_linear_workspace_size(m, 1000, n, kind) == 0


def test_backward_asks_for_what_it_uses():
    """d is there with an epilogue alone, parts of dbias with dbias alone."""
    L = _lib.lib.load()
    m, k, n = 16_384, 32_000, 2048
    size = L.tg_linear_backward_call_workspace_size
    for kind, z in ((F32, 4), (BF16, 2), (F16, 2)):
        assert L.tg_linear_workspace_size(m, n, k, kind) == 0      # (dx, dw: of one part)
        plain, bias = size(m, k, n, kind, 0, 0), size(m, k, n, kind, 0, 1)
        assert plain == 0 and 0 < bias < m * n
        assert size(m, k, n, kind, 3, 0) == m * n * z
        assert size(m, k, n, kind, 3, 1) == m * n * z + bias \
            == L.tg_linear_backward_workspace_size(m, k, n, kind)
    assert size(m, k, n, F32, 9, 0) == size(m, k, n, 7, 0, 0) == size(0, k, n, F32, 0, 0) == 0
