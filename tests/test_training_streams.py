"""How the training operators order the streams that they are called beside: on the host, by a device whose library calls are written down, and on the GPU."""
from types import SimpleNamespace

import pytest
import torch

import localfold_b200 as lf
from localfold_b200 import _native as nat, training
from test_training_refusals import Fake, FakeDevice, float8, weights

T = 1      # torch's current stream


class Device(FakeDevice):
    def __init__(self, log, stream, own=False):
        super().__init__(log, stream)
        answer = lambda name: lambda *args: log.append((name, self.stream) + args[1:2]) or nat.LF_OK      # noqa: E731
        for name in ("lf_float8_decode", "lf_layer_norm_run", "lf_layer_norm_backward_run", "lf_float8_weight_gradient_run"):
            setattr(self.lib, name, answer(name))
        self.lib.lf_float8_linear_workspace = self.lib.lf_layer_norm_backward_workspace = self.lib.lf_float8_weight_gradient_workspace = lambda *sizes: 16
        self._own_stream, self.log = own, log

    def hold(self, tensors):
        self.log.append(("hold", self.stream))


class Memory(Fake):
    """What the operators allocate, too."""

    def new_empty(self, shape, dtype=None):
        count = 1
        for size in shape if isinstance(shape, tuple) else (shape,):
            count *= size
        return Memory(count, dtype or self.dtype)


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(training, "_torch_stream", lambda ordinal: T)
    monkeypatch.setattr(training, "_new", lambda like, dtype, shape: Memory(1, torch.uint8 if dtype == "bytes" else training._torch_dtype(dtype)).new_empty(shape))


def awaits(log):
    return [e[1:3] for e in log if e[0] == "lf_context_await"]


def order(log):
    return [e[0] for e in log]


@pytest.mark.parametrize("own", [False, True])
def test_allocated_memory_waits_for_torch(host, own):
    """A result's memory may have been given back a moment ago and be in use on torch's stream: whoever made the device's stream, it waits."""
    log = []
    d = Device(log, 2, own)
    calls = {
        "encode": lambda: lf.float8_encode(d, Memory(32), 4, 8),
        "decode": lambda: lf.float8_decode(d, float8(4, 8)),
        "linear": lambda: lf.Float8LinearGpu(d).run({"rows": 4, "channels": 8, "outChannels": 6, "activations": float8(4, 8), "weights": mine}),
        "linear, workspace": lambda: lf.Float8LinearGpu(d).run({"rows": 4, "channels": 8, "outChannels": 6, "activations": Memory(32), "weights": mine}, None, Memory(24)),
        "linear, checkpoint": lambda: lf.Float8LinearGpu(d).run({"rows": 4, "channels": 8, "outChannels": 6, "activations": Memory(32), "weights": mine}, {"checkpoint": "e4m3"}, Memory(24)),
        "input gradient": lambda: lf.Float8LinearGpu(d).input_gradient({"rows": 4, "channels": 8, "outChannels": 6, "gradient": float8(4, 6), "weights": mine}),
        "weight gradient": lambda: lf.Float8LinearGpu(d).weight_gradient({"rows": 4, "channels": 8, "outChannels": 6, "gradient": float8(4, 6), "activations": float8(4, 8)}),
        "norm, statistics": lambda: lf.LayerNormGpu(d).run({"rows": 4, "channels": 8, "activations": Memory(32), "scale": Memory(8), "offset": Memory(8)}, {"statistics": True}, Memory(32)),
        "norm, encode": lambda: lf.LayerNormGpu(d).run({"rows": 4, "channels": 8, "activations": Memory(32), "scale": Memory(8), "offset": Memory(8)}, {"encode": "e4m3"}),
        "backward": lambda: lf.LayerNormGpu(d).backward({"rows": 4, "channels": 8, "gradient": Memory(32), "activations": float8(4, 8), "mean": Memory(4), "inverseDeviation": Memory(4),
                                                         "scale": Memory(8)}, None, Memory(32)),
    }
    mine = weights(6, 8)
    mine.device = d
    for name, call in calls.items():
        log.clear()
        call()
        assert awaits(log) == [(2, T)], name
        assert [n.startswith("lf_") and not n.endswith("await") for n in order(log)] == [False, True, False] and order(log)[-1] == "hold", name


def test_memory_of_the_caller_is_ordered_by_the_caller(host):
    """A device on a stream of the caller's, and nothing allocated: no order is imposed (that of the other operators of such a device)."""
    log = []
    d, mine = Device(log, 2), weights(6, 8)
    mine.device = d
    lf.float8_decode(d, float8(4, 8), None, Memory(32, torch.bfloat16))
    lf.Float8LinearGpu(d).run({"rows": 4, "channels": 8, "outChannels": 6, "activations": float8(4, 8), "weights": mine}, None, Memory(24, torch.bfloat16))
    lf.LayerNormGpu(d).run({"rows": 4, "channels": 8, "activations": Memory(32), "scale": Memory(8), "offset": Memory(8)}, None, Memory(32))
    assert awaits(log) == [] and order(log).count("hold") == 3
    here = Device(log, T)
    log.clear()
    lf.float8_decode(here, float8(4, 8))
    assert order(log) == ["lf_float8_decode"]


@pytest.mark.parametrize("current,held", [(2, True), (T, False)])
@pytest.mark.parametrize("what", ["run", "input_gradient", "update"])
def test_memory_of_weights_is_held(host, monkeypatch, what, current, held):
    """Their memory came from the pool of the stream that was torch's current one then, and goes back to it when they are dropped.  Calls that were made with
    the device's stream as the current one are unknown there: the device keeps the memory."""
    log = []
    d, value = Device(log, 2), Memory(48)
    value.shape = (6, 8)

    def used(closed=False):
        mine = weights(6, 8)
        mine.device, mine._origin = d, T
        call, linear = {"rows": 4, "channels": 8, "outChannels": 6, "weights": mine}, lf.Float8LinearGpu(d)
        for _ in range(3):
            if what == "update":
                mine.update(value)
            elif what == "run":
                linear.run({**call, "activations": float8(4, 8)})
            else:
                linear.input_gradient({**call, "gradient": float8(4, 6)})
        if closed:
            d._finalizer = SimpleNamespace(alive=False)      # (a closed device is through)

    monkeypatch.setattr(training, "_torch_stream", lambda ordinal: current)
    used()
    # by the device, with each call, where its stream is not the current one; else when they are dropped
    assert order(log).count("hold") == (1 if held else 3) and order(log)[-1] == "hold"
    log.clear()
    used(closed=True)
    assert order(log).count("hold") == (0 if held else 3)


def test_memory_of_weights_of_one_stream(host, monkeypatch):
    log = []
    d = Device(log, T)
    for capturing in (False, True):
        mine = weights(6, 8)
        mine.device, mine._origin = d, 5 if capturing else T
        monkeypatch.setattr(training, "_capturing", lambda: capturing)
        lf.Float8LinearGpu(d).run({"rows": 4, "channels": 8, "outChannels": 6, "weights": mine, "activations": float8(4, 8)})
        del mine
        assert order(log).count("hold") == 0


@pytest.mark.gpu
def test_weights_dropped_while_they_are_read():
    """Weights made under one stream, multiplied on another behind a queue, and dropped at once; their memory is written again under the first."""
    n = 4096
    stream = torch.cuda.Stream()
    d = lf.Device(0, stream=stream.cuda_stream)
    x8 = lf.float8_encode(d, torch.randn(n, n, device="cuda"), n, n)
    w = torch.randn(n, n, device="cuda")
    linear, call = lf.Float8LinearGpu(d), {"rows": n, "channels": n, "outChannels": n, "activations": x8}
    want = linear.run({**call, "weights": lf.prepare_float8_linear_weights(d, w)})["output"]
    a = torch.randn(n, n, device="cuda")
    for _ in range(5):
        torch.cuda.synchronize()
        mine = lf.prepare_float8_linear_weights(d, w)
        torch.cuda.synchronize()
        d.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(10):
                a = (a @ a) * 1e-2
            got = linear.run({**call, "weights": mine})["output"]
        del mine
        junk = [torch.full((n * n + 4096 * k,), 255, dtype=torch.uint8, device="cuda") for k in (0, 32, 64)]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del junk
    d.close()


OPERATORS = ["encode", "decode", "norm", "backward", "linear", "weight gradient"]


@pytest.mark.gpu
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("name", OPERATORS)
def test_memory_in_use_on_another_stream(name, own):
    """Memory that work on torch's stream still reads is given back, and an operator of a device on a side stream takes it for its result: what was
    read is what the memory held."""
    rows, c = 60000, 256
    side = torch.cuda.Stream()
    d = lf.Device(0) if own else lf.Device(0, stream=side.cuda_stream)
    x, dy = torch.randn(rows, c, device="cuda").bfloat16(), torch.randn(rows, c, device="cuda").bfloat16()
    scale, mean, inverse = torch.ones(c, device="cuda"), torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    x8, linear, norm = lf.float8_encode(d, x, rows, c), lf.Float8LinearGpu(d), lf.LayerNormGpu(d)
    mine = lf.prepare_float8_linear_weights(d, torch.randn(c, c, device="cuda"))
    wide = 4096
    tall = {"rows": 2000, "channels": c, "outChannels": wide, "activations": lf.float8_encode(d, x[:2000], 2000, c), "gradient": torch.randn(2000, wide, device="cuda").bfloat16()}
    shape = {"rows": rows, "channels": c}
    calls = {
        "encode": (lambda: lf.float8_encode(d, x, rows, c).memory, x8.nbytes),
        "decode": (lambda: lf.float8_decode(d, x8), 2 * x.numel()),
        "norm": (lambda: norm.run({**shape, "activations": x, "scale": scale, "offset": scale})["output"], 2 * x.numel()),
        "backward": (lambda: norm.backward({**shape, "activations": x, "gradient": dy, "scale": scale, "mean": mean, "inverseDeviation": inverse})["activations"], 2 * x.numel()),
        "linear": (lambda: linear.run({**shape, "outChannels": c, "activations": x8, "weights": mine})["output"], 2 * x.numel()),
        "weight gradient": (lambda: linear.weight_gradient(tall)["weight"], 4 * wide * c),
    }
    call, size = calls[name]
    d.synchronize()
    torch.cuda.synchronize()
    call()      # (modules are loaded)
    d.synchronize()
    a, total = torch.randn(4096, 4096, device="cuda"), torch.zeros((), dtype=torch.int64, device="cuda")
    met = 0
    for _ in range(5):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        read = torch.full((size,), 3, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for _ in range(20):      # (some ten milliseconds in front of the reader)
            a = (a @ a) * 1e-2
        total = read.sum(dtype=torch.int64)
        place = read.data_ptr()
        del read
        got = call()
        met += got.data_ptr() == place
        torch.cuda.synchronize()
        d.synchronize()
        assert int(total) == 3 * size
        del got
    assert met, "the result never took the memory: this shows nothing"
    d.close()


@pytest.mark.gpu
def test_default_stream_device_beside_a_side_stream():
    """A device on CUDA's default stream, called while torch's current stream is another."""
    d, side = lf.Device(0, stream=0), torch.cuda.Stream()
    x = torch.randn(3000, 256, device="cuda")
    want = lf.float8_decode(d, lf.float8_encode(d, x, 3000, 256), {"output": "f32"})
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(5):
            got = lf.float8_decode(d, lf.float8_encode(d, x, 3000, 256), {"output": "f32"})
            d.synchronize()
            assert torch.equal(got, want)
    d.close()
