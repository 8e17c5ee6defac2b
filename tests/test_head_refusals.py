"""Calls of the dense layers, the log probabilities and the distillation that are
refused before any device work, through the C-ABI and the Python front end,
without a GPU."""
import ctypes as C

import pytest
import torch

from test_expert_refusals import D, N, _Fake, fake, refused
from tinygnn_amd import _lib

I32 = torch.int32


LINEAR = dict(m=10, k=8, n=6, type=0, x=D, ldx=8, w=D, ldw=6, transposed=0, bias=N, act=0,
              residual=N, ldr=0, y=D, ldy=6, pre=N, ldp=0, ws=N, size=0, stream=N)


@pytest.mark.parametrize("change,text", [
    (dict(m=-1), "negative dimension"),
    (dict(k=2 ** 31 - 100), "must be < 2^31 - 4096"),
    (dict(type=3), "unknown element type 3"),
    (dict(act=5), "unknown epilogue 5"),
    (dict(act=-1), "unknown epilogue -1"),
    (dict(x=N), "null pointer"),
    (dict(w=N), "null pointer"),
    (dict(y=N), "null pointer"),
    (dict(ldx=7), "leading dimension below the columns"),
    (dict(ldw=5), "leading dimension below the columns"),
    (dict(transposed=1, ldw=7), "leading dimension below the columns"),
    (dict(ldy=5), "leading dimension below the columns"),
    (dict(residual=D, ldr=5), "leading dimension below the columns"),
    (dict(pre=D, ldp=5), "leading dimension below the columns"),
])
def test_linear(change, text):
    a = dict(LINEAR)
    a.update(change)
    refused("tg_linear", list(a.values()), text)


BACK = dict(m=10, k=8, n=6, type=0, dy=D, lddy=6, x=D, ldx=8, w=D, ldw=6, transposed=0, pre=D,
            ldp=6, act=1, dx=D, lddx=8, dw=D, dbias=D, ws=D, size=1 << 40, stream=N)


@pytest.mark.parametrize("change,text", [
    (dict(n=-1), "negative dimension"),
    (dict(type=-1), "unknown element type -1"),
    (dict(act=7), "unknown epilogue 7"),
    (dict(dy=N), "null pointer"),
    (dict(pre=N), "null pointer"),
    (dict(x=N), "null pointer"),
    (dict(w=N), "null pointer"),
    (dict(lddy=5), "leading dimension below the columns"),
    (dict(ldp=5), "leading dimension below the columns"),
    (dict(ldx=7), "leading dimension below the columns"),
    (dict(ldw=5), "leading dimension below the columns"),
    (dict(lddx=7), "leading dimension below the columns"),
    (dict(size=100), "workspace too small"),
])
def test_linear_backward(change, text):
    a = dict(BACK)
    a.update(change)
    refused("tg_linear_backward", list(a.values()), text)


def test_linear_workspaces():
    L = _lib.lib.load()
    assert L.tg_linear_workspace_size(0, 5, 5, 0) == 0
    assert L.tg_linear_workspace_size(5, 5, 5, 9) == 0
    need = L.tg_linear_workspace_size(100, 8192, 64, 1)
    assert need > 0   # few tiles of a long contraction: cut
    a = dict(LINEAR)
    a.update(m=100, k=8192, n=64, type=1, ldx=8192, ldw=64, ldy=64, ws=D, size=1)
    refused("tg_linear", list(a.values()), "workspace too small")
    # d, dbias' parts, and one product's parts at a time
    assert L.tg_linear_backward_workspace_size(1000, 64, 64, 1) >= 1000 * 64 * 2 + 64 * 4


LOGP = dict(rows=4, classes=9, type=0, logits=D, ld=9, labels=D, temperature=1.0, top=2, value=D,
            entropy=N, top_values=D, top_ids=D, stats=D, ws=N, size=0, stream=N)


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "negative dimension"),
    (dict(classes=0), "no classes"),
    (dict(rows=2 ** 31), "< 2^31"),
    (dict(type=3), "unknown element type 3"),
    (dict(temperature=0.0), "temperature must be between"),
    (dict(temperature=-1.0), "temperature must be between"),
    (dict(temperature=float("nan")), "temperature must be between"),
    (dict(temperature=float("inf")), "temperature must be between"),
    (dict(top=-1), "top must be between"),
    (dict(top=10), "min(64, classes), got 10"),
    (dict(classes=100, ld=100, top=65), "got 65"),
    (dict(ld=8), "leading dimension below classes"),
    (dict(labels=N), "go together"),
    (dict(value=N), "go together"),
    (dict(logits=N), "null pointer"),
    (dict(top_ids=N), "null pointer"),
    (dict(rows=1, classes=200_000, ld=200_000, ws=D, size=64), "workspace too small"),
])
def test_log_probs(change, text):
    a = dict(LOGP)
    a.update(change)
    refused("tg_log_probs", list(a.values()), text)


LOGP_BACK = dict(rows=4, classes=9, type=0, logits=D, ld=9, labels=D, temperature=1.0, stats=D,
                 entropy=D, dvalue=D, dentropy=D, dlogits=D, lddl=9, stream=N)


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "negative dimension"),
    (dict(type=4), "unknown element type 4"),
    (dict(temperature=1e9), "temperature must be between"),
    (dict(lddl=8), "leading dimension below classes"),
    (dict(ld=8), "leading dimension below classes"),
    (dict(dvalue=N), "labels and dvalue go together"),
    (dict(labels=N), "labels and dvalue go together"),
    (dict(entropy=N), "dentropy needs the entropy"),
    (dict(stats=N), "null pointer"),
    (dict(dlogits=N), "null pointer"),
])
def test_log_probs_backward(change, text):
    a = dict(LOGP_BACK)
    a.update(change)
    refused("tg_log_probs_backward", list(a.values()), text)


DISTILL = dict(rows=4, classes=9, k=3, type=0, logits=D, ld=9, teacher_type=1, teacher=D, ids=D,
               temperature=1.0, loss=D, dloss=D, dlogits=D, lddl=9, ws=N, size=0, stream=N)


@pytest.mark.parametrize("change,text", [
    (dict(classes=-1), "negative dimension"),
    (dict(classes=0), "no classes"),
    (dict(type=3), "unknown element type 3"),
    (dict(teacher_type=-2), "unknown element type -2"),
    (dict(k=0), "k must be between 1 and 256, got 0"),
    (dict(k=257), "got 257"),
    (dict(temperature=0.0), "temperature must be between"),
    (dict(ld=8), "leading dimension below classes"),
    (dict(lddl=8), "leading dimension below classes"),
    (dict(dloss=N), "dloss and dlogits go together"),
    (dict(dlogits=N), "dloss and dlogits go together"),
    (dict(teacher=N), "null pointer"),
    (dict(ids=N), "null pointer"),
    (dict(loss=N), "null pointer"),
    (dict(rows=2, classes=900_000, ld=900_000, lddl=900_000, ws=D, size=64),
     "workspace too small"),
])
def test_distill(change, text):
    a = dict(DISTILL)
    a.update(change)
    refused("tg_distill", list(a.values()), text)


def test_loss_workspaces():
    L = _lib.lib.load()
    assert L.tg_log_probs_workspace_size(1, 41, 5, 0) == 0
    assert L.tg_log_probs_workspace_size(0, 500_000, 5, 0) == 0
    assert L.tg_log_probs_workspace_size(1, 500_000, 5, 7) == 0
    # a row of 500,000 is cut: sums and 5 classes of each segment
    assert L.tg_log_probs_workspace_size(1, 500_000, 5, 0) >= 8 * (16 + 5 * 8)
    assert L.tg_distill_workspace_size(3, 500_000, 7, 1) >= 3 * 7 * 4


def test_host_tensors_are_refused():
    import tinygnn_amd as tg
    x, i = torch.zeros(4, 8), torch.zeros(4, dtype=I32)
    r = tg.LogProbs(x[:, 0], None, None, None, torch.zeros(4, 2), 1.0)
    for call in (lambda: tg.linear(x, torch.zeros(8, 3)),
                 lambda: tg.linear_backward(torch.zeros(4, 3), x, torch.zeros(8, 3)),
                 lambda: tg.log_probs(x, i),
                 lambda: tg.log_probs_backward(x[:, 0], x, i, r),
                 lambda: tg.log_probs_backward(None, x, None, r),
                 lambda: tg.distill(x, x[:, :2].contiguous(), i.view(4, 1).repeat(1, 2))):
        with pytest.raises(ValueError, match="expects device"):
            call()


def result(tg, rows=4, entropy=None, temperature=1.0):
    return tg.LogProbs(fake(rows), entropy, None, None, fake(rows, 2), temperature)


@pytest.mark.parametrize("call,text", [
    (lambda tg: tg.linear(fake(4, 8), fake(7, 3)), "dimension mismatch"),
    (lambda tg: tg.linear(fake(4, 8), fake(8, 3), transpose=True), "dimension mismatch"),
    (lambda tg: tg.linear(fake(4, 8), fake(8, 3, dtype=torch.bfloat16)), "w must be"),
    (lambda tg: tg.linear(fake(4, 8), fake(2, 8, 3)), "w must be"),
    (lambda tg: tg.linear(fake(2, 4, 8), fake(8, 3)), "dimension mismatch"),
    (lambda tg: tg.linear(fake(4, 8, dtype=torch.float64), fake(8, 3, dtype=torch.float64)),
     "float32, bfloat16 or float16"),
    (lambda tg: tg.linear(fake(8, 4).t(), fake(8, 3)), "contiguous rows"),
    (lambda tg: tg.linear(fake(4, 8), fake(3, 8).t()), "contiguous rows"),
    (lambda tg: tg.linear(fake(4, 8), fake(8, 3), bias=fake(1, 3)), "bias must be"),
    (lambda tg: tg.linear(fake(4, 8), fake(8, 3), residual=fake(4, 2)), "residual must be"),
    (lambda tg: tg.linear(fake(4, 8), fake(8, 3), out=fake(3, 3)), "out must be"),
    (lambda tg: tg.linear_backward(fake(4, 2), fake(4, 8), fake(8, 3)), "dy must be"),
    (lambda tg: tg.linear_backward(fake(4, 3), fake(4, 8), fake(8, 3), epilogue=tg.EPI_GELU),
     "needs pre"),
    (lambda tg: tg.linear_backward(fake(4, 3), fake(4, 8), fake(8, 3), pre=fake(4, 2),
                                   epilogue=tg.EPI_GELU), "pre must be"),
    (lambda tg: tg.log_probs(fake(4)), "logits must be a matrix"),
    (lambda tg: tg.log_probs(fake(4, 8), fake(4)), "labels must be"),
    (lambda tg: tg.log_probs(fake(4, 8), fake(3, dtype=I32)), "labels must be"),
    (lambda tg: tg.log_probs(fake(4, 8), top=9), "top must be between"),
    (lambda tg: tg.log_probs(fake(4, 100), top=65), "top must be between"),
    (lambda tg: tg.log_probs_backward(fake(4), fake(4, 8), None, result(tg)), "go together"),
    (lambda tg: tg.log_probs_backward(None, fake(4, 8), fake(4, dtype=I32), result(tg)),
     "go together"),
    (lambda tg: tg.log_probs_backward(fake(3), fake(4, 8), fake(4, dtype=I32), result(tg)),
     "dvalue must be"),
    (lambda tg: tg.log_probs_backward(fake(4), fake(4, 8), fake(4, dtype=I32), result(tg, 3)),
     "stats must be"),
    (lambda tg: tg.log_probs_backward(fake(4), fake(4, 8), fake(4, dtype=I32), result(tg),
                                      dentropy=fake(4)), "needs log_probs' entropy"),
    (lambda tg: tg.log_probs_backward(fake(4), fake(4, 8), fake(4, dtype=I32), result(tg),
                                      temperature=2.0), "temperature 2.0 is not"),
    (lambda tg: tg.log_probs_backward(fake(4), fake(4, 8), fake(4, dtype=I32), result(tg),
                                      out=fake(4, 7)), "out must be"),
    (lambda tg: tg.distill(fake(4, 8), fake(3, 2), fake(3, 2, dtype=I32)), "teacher must be"),
    (lambda tg: tg.distill(fake(4, 8), fake(4, 0), fake(4, 0, dtype=I32)), "teacher must be"),
    (lambda tg: tg.distill(fake(4, 8), fake(4, 257), fake(4, 257, dtype=I32)), "teacher must be"),
    (lambda tg: tg.distill(fake(4, 8), fake(4, 2), fake(4, 2)), "ids must be"),
    (lambda tg: tg.distill(fake(4, 8), fake(4, 2, dtype=torch.float64), fake(4, 2, dtype=I32)),
     "float32, bfloat16 or float16"),
    (lambda tg: tg.distill(fake(4, 8), fake(4, 2), fake(4, 2, dtype=I32), dloss=fake(3)),
     "dloss must be"),
    (lambda tg: tg.distill(fake(4, 8), fake(4, 2), fake(4, 2, dtype=I32), out=fake(4, 8)),
     "needs dloss"),
])
def test_shapes_are_refused(monkeypatch, call, text):
    import tinygnn_amd as tg
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    names = tg._Torch()
    names.raw_stream = lambda index: 0
    monkeypatch.setattr(tg, "_pt", names)
    with pytest.raises(tg.InvalidArgument, match=text):
        call(tg)


class _Other(_Fake):
    device = torch.device("cuda", 1)

    def get_device(self):
        return 1


def test_two_devices_are_refused(monkeypatch):
    import tinygnn_amd as tg
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    names = tg._Torch()
    names.raw_stream = lambda index: 0
    monkeypatch.setattr(tg, "_pt", names)
    with pytest.raises(tg.InvalidArgument, match="tensors on cuda:0 and cuda:1"):
        tg.linear(fake(4, 8), torch.zeros(8, 3).as_subclass(_Other))
    with pytest.raises(tg.InvalidArgument, match="tensors on cuda:0 and cuda:1"):
        tg.distill(fake(4, 8), fake(4, 2), torch.zeros(4, 2, dtype=I32).as_subclass(_Other))


# ---------------------------------------------------------------------------
# A stream that is not the current one runs after it
# ---------------------------------------------------------------------------
CALLS = {
    "linear": lambda tg, d, s: tg.linear(d(4, 8), d(8, 3), stream=s),
    "linear_backward": lambda tg, d, s: tg.linear_backward(d(4, 3), d(4, 8), d(8, 3), stream=s),
    "log_probs": lambda tg, d, s: tg.log_probs(d(4, 8), d(4, dtype=I32), top=2, stream=s),
    "log_probs_backward": lambda tg, d, s: tg.log_probs_backward(
        d(4), d(4, 8), d(4, dtype=I32), tg.LogProbs(d(4), None, None, None, d(4, 2), 1.0),
        stream=s),
    "distill": lambda tg, d, s: tg.distill(d(4, 8), d(4, 2), d(4, 2, dtype=I32), dloss=d(4),
                                           stream=s),
}


@pytest.mark.parametrize("name", list(CALLS))
@pytest.mark.parametrize("kind", ["torch", "handle", "current"])
def test_waits_for_the_current_stream(monkeypatch, name, kind):
    import test_stream_order as order
    import tinygnn_amd as tg
    current = order._Queue(5)
    stream = dict(torch=order._Queue(77), handle=order._Handle(77), current=current)[kind]
    made, seen = [], []
    current.queue.append(lambda: made.append(True))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: current)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    names = tg._Torch()
    names.raw_stream = lambda index: 5
    names.empty = lambda shape, dtype=None, device=None: torch.empty(shape, dtype=dtype)
    monkeypatch.setattr(tg, "_pt", names)
    monkeypatch.setattr(tg, "lib", order._Lib(made, seen))
    CALLS[name](tg, order.dev, stream)
    assert seen == [(stream.cuda_stream, kind != "current")]
    assert bool(current.queue) == (kind == "current")
