"""Calls of the expert-layer operators that are refused before any device work,
through the C-ABI and the Python front end, without a GPU."""
import ctypes as C

import pytest
import torch

from tinygnn_amd import _lib

D = C.c_void_p(16)   # a pointer that is never followed: the calls fail on the host
N = None


def refused(name, args, text):
    L = _lib.lib.load()
    assert getattr(L, name)(*args) == _lib.TG_ERR_INVALID_ARGUMENT, name
    assert text in L.tg_last_error().decode(), L.tg_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "negative dimension"),
    (dict(cols=0), "no mean"),
    (dict(type=3), "unknown element type 3"),
    (dict(wtype=2), "gamma and beta must have x's type or be floats"),
    (dict(x=N), "null pointer"),
    (dict(ldx=7), "leading dimension below cols"),
    (dict(rows=2 ** 31), "< 2^31"),
])
def test_layer_norm(change, text):
    a = dict(rows=4, cols=8, type=1, x=D, ldx=8, gamma=D, beta=D, wtype=1, eps=1e-5, y=D, ldy=8)
    a.update(change)
    refused("tg_layer_norm", [*a.values(), N, N, N], text)
    back = [a["rows"], a["cols"], a["type"], D, 8, a["x"], a["ldx"], D, a["wtype"], D, D, D, 8, D,
            D, D, 1 << 40, N]
    refused("tg_layer_norm_backward", back, text)


def test_layer_norm_backward_workspace():
    L = _lib.lib.load()
    need = L.tg_layer_norm_backward_workspace_size(1000, 64)
    assert need >= 2 * 64 * 4 and L.tg_layer_norm_backward_workspace_size(0, 64) == 0
    refused("tg_layer_norm_backward",
            [1000, 64, 0, D, 64, D, 64, D, 0, D, D, D, 64, D, D, D, need - 1, N],
            "workspace too small")


@pytest.mark.parametrize("tokens,experts,k,type,ld,text", [
    (-1, 4, 2, 0, 4, "negative dimension"),
    (5, 0, 1, 0, 4, "between 1 and 1024 experts"),
    (5, 1025, 1, 0, 1025, "between 1 and 1024 experts"),
    (5, 4, 5, 0, 4, "k must be between 1 and min(32, experts), got 5"),
    (5, 64, 33, 0, 64, "got 33"),
    (5, 4, 0, 0, 4, "got 0"),
    (2 ** 30, 4, 2, 0, 4, "tokens * k must be < 2^31"),
    (5, 4, 2, 0, 3, "leading dimension below experts"),
    (5, 4, 2, 9, 4, "unknown element type 9"),
])
def test_route(tokens, experts, k, type, ld, text):
    refused("tg_route", [tokens, experts, k, type, D, ld, 0, D, D, D, D, D, D, 1 << 40, N], text)
    refused("tg_route_backward", [tokens, experts, k, type, D, ld, 0, D, D, D, D, 1 << 20, N],
            text)


def test_route_pointers():
    ok = [5, 4, 2, 0, D, 4, 0, D, D, D, D, D, N, 0, N]
    for at in (4, 7, 8):
        refused("tg_route", ok[:at] + [N] + ok[at + 1:], "null pointer")
    for at in (9, 10, 11):
        refused("tg_route", ok[:at] + [N] + ok[at + 1:], "go together")
    L = _lib.lib.load()
    need = L.tg_route_workspace_size(100_000, 64, 2)
    refused("tg_route", [100_000, 64, 2, 0, D, 64, 0, D, D, D, D, D, D, need - 256, N],
            "workspace too small")
    assert L.tg_route_workspace_size(8, 64, 2) == 0


@pytest.mark.parametrize("n,groups,k,text", [(-1, 4, 1, "n must be"), (2 ** 31, 4, 1, "n must be"),
                                             (5, 0, 1, "groups, got 0"),
                                             (5, 1025, 1, "groups, got 1025"), (5, 4, 0, "k must")])
def test_route_plan(n, groups, k, text):
    refused("tg_route_plan", [n, groups, k, D, D, D, D, D, 1 << 40, N], text)


@pytest.mark.parametrize("tokens,k,cols,type,ld,text", [
    (-1, 2, 4, 0, 4, "negative dimension"),
    (2 ** 30, 2, 4, 0, 4, "must be < 2^31"),
    (3, 2, 4, 0, 3, "leading dimension below cols"),
    (3, 2, 4, -1, 4, "unknown element type -1"),
])
def test_combine(tokens, k, cols, type, ld, text):
    refused("tg_route_combine", [tokens, k, cols, type, D, 9, ld, D, D, D, ld, N], text)
    refused("tg_route_combine_backward",
            [tokens, k, cols, type, D, ld, D, 9, ld, D, D, D, ld, D, N], text)


@pytest.mark.parametrize("change,text", [
    (dict(m=-1), "negative dimension"),
    (dict(m=2 ** 31 - 100), "must be < 2^31 - 4096"),
    (dict(groups=1025), "at most 1024 groups, got 1025"),
    (dict(type=7), "unknown element type 7"),
    (dict(x_rows=9), "x has fewer than m rows"),
    (dict(offsets=N), "null pointer"),
    (dict(ldx=7), "leading dimension below the columns"),
])
def test_grouped(change, text):
    a = dict(m=10, k=8, n=6, groups=2, type=0, x=D, x_rows=10, ldx=8, rows=N, offsets=D)
    a.update(change)
    refused("tg_grouped_matmul", [*a.values(), D, 6, 48, 0, N, 0, D, 6, N], text)
    refused("tg_grouped_matmul_wgrad",
            [*list(a.values())[:9], D, 6, a["offsets"], D, D, D, 1 << 50, N], text)


def test_grouped_epilogue_and_weights():
    a = [10, 8, 6, 2, 0, D, 10, 8, N, D, D]
    refused("tg_grouped_matmul", [*a, 6, 48, 0, N, 3, D, 6, N], "unknown epilogue 3")
    refused("tg_grouped_matmul", [*a, 5, 48, 0, N, 0, D, 6, N], "leading dimension")
    refused("tg_grouped_matmul", [*a, 7, 48, 1, N, 0, D, 6, N], "leading dimension")
    refused("tg_grouped_matmul", [*a, 6, 48, 0, N, 0, N, 6, N], "null pointer")


@pytest.mark.parametrize("change,text", [
    (dict(k=-1), "negative dimension"),
    (dict(groups=2), "several groups need offsets"),
    (dict(groups=1025, offsets=D), "at most 1024 groups"),
    (dict(x_rows=3), "x has fewer than m rows"),
    (dict(type=4), "unknown element type 4"),
    (dict(epi=-1), "unknown epilogue -1"),
    (dict(ldy=5), "leading dimension"),
    (dict(xq=C.c_void_p(24)), "16-byte aligned"),
    (dict(wq=C.c_void_p(24)), "16-byte aligned"),
    (dict(wscale=N), "null pointer"),
])
def test_matmul_fp8(change, text):
    a = dict(m=10, k=8, n=6, groups=1, xq=D, xscale=D, x_rows=10, rows=N, offsets=N, wq=D,
             wscale=D, type=1, bias=N, epi=0, y=D, ldy=6)
    a.update(change)
    refused("tg_matmul_fp8", [*a.values(), N], text)


def test_quantize():
    refused("tg_quantize", [-1, 8, 0, D, 8, D, D, N], "negative dimension")
    refused("tg_quantize", [3, 8, 0, D, 7, D, D, N], "leading dimension")
    refused("tg_quantize", [3, 8, 0, D, 8, C.c_void_p(4), D, N], "16-byte aligned")
    refused("tg_quantize", [3, 8, 3, D, 8, D, D, N], "unknown element type 3")
    refused("tg_quantize_weight", [1025, 8, 8, 0, D, 8, 64, 0, D, D, N], "at most 1024 groups")
    refused("tg_quantize_weight", [1, 8, 6, 0, D, 7, 64, 1, D, D, N], "leading dimension")
    refused("tg_quantize_weight", [1, 8, 6, 0, D, 8, 64, 0, N, D, N], "null pointer")


def test_host_tensors_are_refused():
    import tinygnn_amd as tg
    x = torch.zeros(4, 8)
    off = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: tg.layer_norm(x), lambda: tg.route(x, 2),
                 lambda: tg.route_plan(off, 2), lambda: tg.quantize(x),
                 lambda: tg.route_combine(x, off.view(-1, 1)),
                 lambda: tg.grouped_matmul(x, torch.zeros(2, 8, 3), off),
                 lambda: tg.grouped_matmul_wgrad(x, x, off)):
        with pytest.raises(ValueError, match="expects device"):
            call()


class _Fake(torch.Tensor):
    """A host tensor that says it is on the GPU: shape and type checks come
    before anything touches a device."""
    is_cuda = True
    device = torch.device("cuda", 0)

    def get_device(self):
        return 0


def fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Fake)


I32 = torch.int32


@pytest.mark.parametrize("call,text", [
    (lambda tg: tg.layer_norm(fake(4)), "x must be a matrix"),
    (lambda tg: tg.layer_norm(fake(4, 8, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (lambda tg: tg.layer_norm(fake(8, 4).t()), "contiguous rows"),
    (lambda tg: tg.layer_norm(fake(4, 8), fake(7)), "gamma must be"),
    (lambda tg: tg.layer_norm(fake(4, 8), fake(8), fake(8, dtype=torch.float16)), "beta must be"),
    (lambda tg: tg.layer_norm(fake(4, 8), out=fake(4, 7)), "out must be"),
    (lambda tg: tg.layer_norm_backward(fake(4, 7), fake(4, 8), fake(4), fake(4)), "dy must be"),
    (lambda tg: tg.layer_norm_backward(fake(4, 8), fake(4, 8), fake(3), fake(4)), "mean must be"),
    (lambda tg: tg.route(fake(4, 8), 9), "k must be between"),
    (lambda tg: tg.route_plan(fake(4), 3), "int32"),
    (lambda tg: tg.route_plan(fake(4, dtype=I32), 0), "1024 groups"),
    (lambda tg: tg.route_backward(fake(4, 2), fake(4, 8), fake(4, 3), fake(4, 3, dtype=I32)),
     "dweights must be"),
    (lambda tg: tg.route_combine(fake(4, 8), fake(2, 2, dtype=torch.int64)), "position must be"),
    (lambda tg: tg.route_combine(fake(4, 8), fake(2, 2, dtype=I32), fake(2, 3)), "weights must"),
    (lambda tg: tg.grouped_matmul(fake(4, 8), fake(2, 7, 3), fake(3, dtype=I32)),
     "dimension mismatch"),
    (lambda tg: tg.grouped_matmul(fake(4, 8), fake(3, 8, 3), fake(3, dtype=I32)), "w must be"),
    (lambda tg: tg.grouped_matmul(fake(4, 8), fake(2, 3, 8).transpose(1, 2), fake(3, dtype=I32)),
     "contiguous rows"),
    (lambda tg: tg.grouped_matmul(fake(4, 8), fake(2, 8, 3), fake(3)), "offsets must be"),
    (lambda tg: tg.grouped_matmul(fake(4, 8), fake(2, 8, 3), fake(3, dtype=I32), bias=fake(3)),
     "bias must be"),
    (lambda tg: tg.grouped_matmul_wgrad(fake(4, 8), fake(5, 3), fake(3, dtype=I32)),
     "dy must be"),
    (lambda tg: tg.quantize_weight(fake(8)), "w must be"),
    (lambda tg: tg.matmul_fp8(tg.BlockRows(fake(4, 128), fake(1, 4), 8),
                              tg.BlockWeight(fake(3, 128), fake(1, 1), 9)), "dimension mismatch"),
    (lambda tg: tg.matmul_fp8(tg.BlockRows(fake(4, 64), fake(1, 4), 8),
                              tg.BlockWeight(fake(3, 128), fake(1, 1), 8)), "x.q must be"),
])
def test_shapes_are_refused(monkeypatch, call, text):
    import tinygnn_amd as tg
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    names = tg._Torch()
    names.raw_stream = lambda index: 0
    monkeypatch.setattr(tg, "_pt", names)
    with pytest.raises(tg.InvalidArgument, match=text):
        call(tg)
