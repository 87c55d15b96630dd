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
