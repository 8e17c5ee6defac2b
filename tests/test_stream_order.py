"""Calls on an explicit stream that is not torch's current one run after what
is queued on the current one: what makes their inputs, and what the last holders
of their outputs' memory still do.

Without a GPU a stream is a queue, and `wait_stream` runs the other's: a call
that does not wait reads its input too early every time.  With one, the calls
follow a long queue on the current stream."""
import pytest
import torch

from expert_cases import gen, randn


class _Queue:
    """A stream whose work runs when another stream, or the host, waits."""

    def __init__(self, handle):
        self.cuda_stream, self.queue = handle, []

    def synchronize(self):
        while self.queue:
            self.queue.pop(0)()

    def wait_stream(self, other):
        other.synchronize()


class _Handle:
    """A stream of another library: a handle to wait for, and no more."""

    def __init__(self, handle):
        self.cuda_stream = handle

    def synchronize(self):
        pass


class _Device(torch.Tensor):
    """A host tensor that says it is on the GPU."""
    is_cuda = True
    device = torch.device("cuda", 0)

    def get_device(self):
        return 0


def dev(*shape, dtype=torch.float32):
    return torch.ones(*shape, dtype=dtype).as_subclass(_Device)


class _Lib:
    """Native calls that note the stream and whether the work before was done."""

    def __init__(self, made, seen):
        self.made, self.seen = made, seen

    def check(self, status):
        assert status == 0

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_size"):
                return 16
            self.seen.append((args[-1], bool(self.made)))
            return 0
        return call


I32 = torch.int32


def block_rows(tg):
    return tg.BlockRows(dev(4, 128, dtype=torch.float8_e4m3fn), dev(1, 4), 8)


CALLS = {
    "matmul": lambda tg, s: tg.matmul(dev(4, 8), dev(8, 3), out=dev(4, 3), stream=s),
    "softmax": lambda tg, s: tg.softmax_(dev(4, 8), stream=s),
    "spmm": lambda tg, s: tg.spmm(tg.DeviceCSR(2, 4, dev(3, dtype=I32), dev(2, dtype=I32), dev(2)),
                                  dev(4, 8), out=dev(2, 8), stream=s),
    "layer_norm": lambda tg, s: tg.layer_norm(dev(4, 8), stream=s),
    "layer_norm_backward": lambda tg, s: tg.layer_norm_backward(dev(4, 8), dev(4, 8), dev(4),
                                                                dev(4), stream=s),
    "route": lambda tg, s: tg.route(dev(4, 8), 2, stream=s),
    "route_plan": lambda tg, s: tg.route_plan(dev(4, dtype=I32), 3, stream=s),
    "route_backward": lambda tg, s: tg.route_backward(dev(4, 2), dev(4, 8), dev(4, 2),
                                                      dev(4, 2, dtype=I32), stream=s),
    "route_combine": lambda tg, s: tg.route_combine(dev(8, 3), dev(4, 2, dtype=I32), stream=s),
    "route_combine_backward": lambda tg, s: tg.route_combine_backward(
        dev(4, 3), dev(8, 3), dev(4, 2, dtype=I32), stream=s),
    "grouped_matmul": lambda tg, s: tg.grouped_matmul(dev(4, 8), dev(2, 8, 3),
                                                      dev(3, dtype=I32), stream=s),
    "grouped_matmul_wgrad": lambda tg, s: tg.grouped_matmul_wgrad(
        dev(4, 8), dev(4, 3), dev(3, dtype=I32), stream=s),
    "quantize": lambda tg, s: tg.quantize(dev(4, 8), stream=s),
    "quantize_weight": lambda tg, s: tg.quantize_weight(dev(8, 3), stream=s),
    "matmul_fp8": lambda tg, s: tg.matmul_fp8(
        block_rows(tg), tg.BlockWeight(dev(3, 128, dtype=torch.float8_e4m3fn), dev(1, 1), 8),
        stream=s),
}


@pytest.mark.parametrize("name", list(CALLS))
@pytest.mark.parametrize("kind", ["torch", "handle", "current"])
def test_waits_for_the_current_stream(monkeypatch, name, kind):
    import tinygnn_amd as tg
    current = _Queue(5)
    stream = dict(torch=_Queue(77), handle=_Handle(77), current=current)[kind]
    made, seen = [], []
    current.queue.append(lambda: made.append(True))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: current)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    names = tg._Torch()
    names.raw_stream = lambda index: 5
    names.empty = lambda shape, dtype=None, device=None: torch.empty(shape, dtype=dtype)
    monkeypatch.setattr(tg, "_pt", names)
    monkeypatch.setattr(tg, "dptr", lambda t, dtype=None: 16)
    monkeypatch.setattr(tg, "lib", _Lib(made, seen))
    CALLS[name](tg, stream)
    # on the current stream the order is there, and nothing waits
    assert seen == [(stream.cuda_stream, kind != "current")]
    assert bool(current.queue) == (kind == "current")


def _late(value):
    """An input of `value` that some milliseconds of work on the current stream
    come before."""
    x = torch.zeros_like(value)
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(10):
        big = torch.mm(big, big)
    x.copy_(value)
    return x


@pytest.mark.gpu
def test_inputs_of_the_current_stream(gpu):
    import tinygnn_amd as tg
    side, g = torch.cuda.Stream(), gen(1)
    value, w = randn(g, (700, 96), torch.float32), randn(g, (4, 96, 40), torch.float32)
    off = torch.tensor([0, 100, 100, 600, 700], dtype=torch.int32, device="cuda")
    for call in (lambda x, s: tg.layer_norm(x, stream=s),
                 lambda x, s: tg.route(x, 3, stream=s)[0],
                 lambda x, s: tg.grouped_matmul(x, w, off, stream=s),
                 lambda x, s: tg.grouped_matmul_wgrad(x, x, off, stream=s)[0],
                 lambda x, s: tg.quantize(x, stream=s).scale):
        want = call(value, None)
        assert torch.equal(call(_late(value), side), want)
    a = tg.matmul(value, w[0])
    out = torch.empty_like(a)
    tg.matmul(_late(value), w[0], out=out, stream=side)
    side.synchronize()
    assert torch.equal(out, a)


@pytest.mark.gpu
def test_memory_of_the_current_stream(gpu):
    """A block that was dropped with work on it still queued becomes the call's
    output: that work comes first."""
    import tinygnn_amd as tg
    side = torch.cuda.Stream()
    x = randn(gen(2), (1 << 14, 256), torch.float32)
    want = tg.layer_norm(x)
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    held = [torch.empty_like(x) for _ in range(16)]   # what the allocator may have kept, too
    places = {t.data_ptr() for t in held}
    torch.cuda.synchronize()
    for _ in range(10):
        big = torch.mm(big, big)
    for t in held:
        t.fill_(7.0)
    del held, t
    y = tg.layer_norm(x, stream=side)
    assert y.data_ptr() in places, "the allocator gave another block"
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.gpu
def test_stream_under_capture(gpu):
    """A stream that is being captured waits for nothing: the call is recorded,
    and runs where the graph is launched."""
    import tinygnn_amd as tg
    g = gen(3)
    a, b = randn(g, (300, 64), torch.float32), randn(g, (64, 48), torch.float32)
    want, out = tg.matmul(a, b), torch.zeros(300, 48, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph.capture_begin(capture_error_mode="relaxed")
    tg.matmul(a, b, out=out, stream=side)
    with torch.cuda.stream(side):
        graph.capture_end()
    torch.cuda.synchronize()
    assert not out.any()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
