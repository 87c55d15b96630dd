"""What the training operators refuse, on the host: no GPU and no library call is needed for any of it."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import localfold_b200 as lf
from localfold_b200 import _native as nat, training
from localfold_b200.operators import RangeError


class Fake:
    """Stands where a CUDA tensor does, as far as the checks look."""

    def __init__(self, count, dtype=torch.float32, gpu=0, contiguous=True):
        self.count, self.dtype, self.gpu, self.contiguous, self.is_cuda = count, dtype, gpu, contiguous, True
        self.device, self.shape = torch.device("cuda", gpu), (count,)

    def get_device(self):
        return self.gpu

    def numel(self):
        return self.count

    def is_contiguous(self):
        return self.contiguous

    def element_size(self):
        return 1 if self.dtype == torch.uint8 else 4

    def data_ptr(self):
        return 4096


DEVICE = SimpleNamespace(ordinal=0)


def float8(rows, channels, name="e4m3", gpu=0):
    return lf.Float8Tensor(rows, channels, name, Fake(sum(training._sizes(rows, channels)), torch.uint8, gpu))


def norm_input(**changes):
    return {**{"rows": 4, "channels": 8, "activations": Fake(32, torch.bfloat16), "scale": Fake(8), "offset": Fake(8)}, **changes}


@pytest.mark.parametrize("changes,options,error,text", [
    ({"rows": 0}, None, RangeError, "rows must be a positive safe integer"),
    ({"channels": 2.5}, None, RangeError, "channels must be a positive safe integer"),
    ({"activations": Fake(31, torch.bfloat16)}, None, RangeError, "activations has 31 values; expected 32"),
    ({"activations": torch.zeros(32)}, None, ValueError, "activations must be a CUDA tensor"),
    ({"activations": np.zeros(32, np.float32)}, None, ValueError, "activations must be a CUDA tensor"),
    ({"activations": Fake(32, torch.float16)}, None, ValueError, "activations must be f32 or bf16"),
    ({"activations": Fake(32, gpu=1)}, None, ValueError, "activations is on cuda:1"),
    ({"activations": Fake(32, contiguous=False)}, None, ValueError, "activations must be contiguous"),
    ({"scale": Fake(8, torch.bfloat16)}, None, ValueError, "scale must be f32"),
    ({"offset": Fake(7)}, None, RangeError, "offset has 7 values; expected 8"),
    ({"rows": 2 ** 31}, None, RangeError, "rows must be at most 2147483647; received 2147483648"),
    ({"rows": 1, "channels": 2 ** 40, "activations": Fake(2 ** 40)}, None, RangeError, "channels must be at most 2147483647"),
    ({"epsilon": 1e39}, None, RangeError, "epsilon must be finite and positive"),
    ({"epsilon": float("inf")}, None, RangeError, "epsilon must be finite and positive"),
    ({"epsilon": 0.0}, None, RangeError, "epsilon must be finite and positive"),
    ({"epsilon": float("nan")}, None, RangeError, "epsilon must be finite and positive"),
    ({}, {"checkpoint": "int8"}, ValueError, 'checkpoint must be "e4m3" or "e5m2"'),
    ({}, {"encode": True}, ValueError, 'encode must be "e4m3" or "e5m2"'),
    ({}, {"variance": "none"}, ValueError, "variance"),
])
def test_layer_norm(changes, options, error, text):
    with pytest.raises(error, match=text):
        lf.LayerNormGpu(DEVICE).run(norm_input(**changes), options)


def test_layer_norm_outputs():
    with pytest.raises(ValueError, match="an encoded output is a new Float8Tensor"):
        lf.LayerNormGpu(DEVICE).run(norm_input(), {"encode": "e4m3"}, out=Fake(32, torch.bfloat16))
    with pytest.raises(ValueError, match="out must be bf16"):
        lf.LayerNormGpu(DEVICE).run(norm_input(), None, out=Fake(32))


@pytest.mark.parametrize("changes,error,text", [
    ({"gradient": Fake(30, torch.bfloat16)}, RangeError, "gradient has 30 values; expected 32"),
    ({"activations": Fake(32)}, ValueError, "activations must be bf16"),
    ({"activations": float8(4, 9)}, RangeError, "activations is 4 x 9; expected 4 x 8"),
    ({"activations": float8(4, 8, gpu=1)}, ValueError, "activations is on cuda:1"),
    ({"mean": Fake(3)}, RangeError, "mean has 3 values; expected 4"),
    ({"inverseDeviation": Fake(4, torch.bfloat16)}, ValueError, "inverseDeviation must be f32"),
    ({"scale": Fake(9)}, RangeError, "scale has 9 values; expected 8"),
])
def test_layer_norm_backward(changes, error, text):
    good = {"rows": 4, "channels": 8, "gradient": Fake(32, torch.bfloat16), "activations": Fake(32, torch.bfloat16), "mean": Fake(4),
            "inverseDeviation": Fake(4), "scale": Fake(8)}
    with pytest.raises(error, match=text):
        lf.LayerNormGpu(DEVICE).backward({**good, **changes})


def test_float8():
    with pytest.raises(RangeError, match="rows must be a positive safe integer"):
        lf.float8_encode(DEVICE, Fake(8), 0, 8)
    with pytest.raises(RangeError, match="channels must be at most 2147483647"):
        lf.float8_encode(DEVICE, Fake(2 ** 33), 1, 2 ** 33)
    with pytest.raises(ValueError, match='format must be "e4m3" or "e5m2"'):
        lf.float8_encode(DEVICE, Fake(8), 1, 8, {"format": "e3m4"})
    with pytest.raises(RangeError, match="activations has 8 values; expected 16"):
        lf.float8_encode(DEVICE, Fake(8), 2, 8)
    with pytest.raises(ValueError, match="encoded must be a Float8Tensor"):
        lf.float8_decode(DEVICE, Fake(8))
    with pytest.raises(ValueError, match='output must be "f32" or "bf16"'):
        lf.float8_decode(DEVICE, float8(2, 8), {"output": "f16"})
    with pytest.raises(ValueError, match="out must be bf16"):
        lf.float8_decode(DEVICE, float8(2, 8), None, Fake(16))
    with pytest.raises(RangeError, match="memory has 5 values"):
        lf.Float8Tensor(2, 8, "e4m3", Fake(5, torch.uint8))
    with pytest.raises(ValueError, match="memory must be a contiguous uint8 CUDA tensor"):
        lf.Float8Tensor(2, 8, "e4m3", Fake(544))
    with pytest.raises(ValueError, match='format must be "e4m3" or "e5m2"'):
        lf.Float8Tensor(2, 8, "fp8", Fake(544, torch.uint8))


def weights(n, c, gpu=0):
    w = object.__new__(lf.Float8LinearWeights)
    w.device, w.out_channels, w.channels, w.bias = SimpleNamespace(ordinal=gpu) if gpu else DEVICE, n, c, None
    w.forward, w.transposed = float8(n, c), float8(c, n)
    return w


@pytest.mark.parametrize("changes,options,error,text", [
    ({"outChannels": 0}, None, RangeError, "outChannels must be a positive safe integer"),
    ({"outChannels": 7}, None, RangeError, "weights are 6 x 8; expected 7 x 8"),
    ({"channels": 9}, None, RangeError, "weights are 6 x 8; expected 6 x 9"),
    ({"weights": Fake(48)}, None, ValueError, "weights must come from prepare_float8_linear_weights"),
    ({"weights": weights(6, 8, gpu=1)}, None, ValueError, "weights are on cuda:1"),
    ({"activations": Fake(31)}, None, RangeError, "activations has 31 values; expected 32"),
    ({"activations": float8(5, 8)}, None, RangeError, "activations is 5 x 8; expected 4 x 8"),
    ({}, {"format": "e2m1"}, ValueError, 'format must be "e4m3" or "e5m2"'),
    ({}, {"output": "f64"}, ValueError, 'output must be "f32" or "bf16"'),
])
def test_linear(changes, options, error, text):
    good = {"rows": 4, "channels": 8, "outChannels": 6, "activations": Fake(32), "weights": weights(6, 8)}
    with pytest.raises(error, match=text):
        lf.Float8LinearGpu(DEVICE).run({**good, **changes}, options)


class FakeDevice:
    """A device whose library calls are written down."""

    def __init__(self, log, stream):
        self.ordinal, self.stream, self.handle, self._own_stream, self._finalizer = 0, stream, stream, False, SimpleNamespace(alive=True)
        answer = lambda name: lambda *args: log.append((name, self.stream) + args[1:2]) or nat.LF_OK
        self.lib = SimpleNamespace(**{name: answer(name) for name in ("lf_context_await", "lf_float8_encode", "lf_float8_linear_run")})

    def check(self, status):
        assert status == nat.LF_OK

    def hold(self, tensors):
        pass


def test_weights_of_another_device(monkeypatch):
    """Calls wait for the weights' device, a later update for the calls; a device that was closed is not waited for."""
    monkeypatch.setattr(training, "_torch_stream", lambda ordinal: 1)
    log = []
    owner, user = FakeDevice(log, 1), FakeDevice(log, 2)
    w = weights(6, 8)
    w.device, value = owner, Fake(48)
    value.shape = (6, 8)
    call = {"rows": 4, "channels": 8, "outChannels": 6, "activations": float8(4, 8), "weights": w}
    out = Fake(24, torch.bfloat16)
    names = lambda: [e[:3] if e[0] == "lf_context_await" else e[:2] for e in log]
    lf.Float8LinearGpu(user).run(call, None, out)
    w.update(value)
    assert names() == [("lf_context_await", 2, 1), ("lf_float8_linear_run", 2), ("lf_context_await", 1, 2), ("lf_float8_encode", 1)]
    log.clear()
    w.update(value)      # (nothing has read since)
    lf.Float8LinearGpu(owner).run(call, None, out)
    w.update(value)
    assert names() == [("lf_float8_encode", 1), ("lf_float8_linear_run", 1), ("lf_float8_encode", 1)]
    log.clear()
    lf.Float8LinearGpu(user).run(call, None, out)
    user._finalizer.alive = False
    w.update(value)
    user._finalizer.alive, owner._finalizer.alive = True, False
    lf.Float8LinearGpu(user).run(call, None, out)
    assert names() == [("lf_context_await", 2, 1), ("lf_float8_linear_run", 2), ("lf_float8_encode", 1), ("lf_float8_linear_run", 2)]


def test_linear_gradients():
    linear = lf.Float8LinearGpu(DEVICE)
    good = {"rows": 4, "channels": 8, "outChannels": 6, "weights": weights(6, 8)}
    with pytest.raises(RangeError, match="gradient has 32 values; expected 24"):
        linear.input_gradient({**good, "gradient": Fake(32)})
    with pytest.raises(ValueError, match="activations must be a Float8Tensor"):
        linear.weight_gradient({**good, "gradient": Fake(24, torch.bfloat16), "activations": Fake(32)})
    with pytest.raises(ValueError, match="gradient must be bf16"):
        linear.weight_gradient({**good, "gradient": Fake(24), "activations": float8(4, 8)})
    with pytest.raises(RangeError, match="gradient is 4 x 8; expected 4 x 6"):
        linear.weight_gradient({**good, "gradient": float8(4, 8), "activations": float8(4, 8)})
    with pytest.raises(RangeError, match="weight must be"):
        lf.prepare_float8_linear_weights(DEVICE, Fake(48))


def test_library_without_a_context():
    """Every entry point answers a null context with a status, every size function with none or a size."""
    lib, res = nat.load(), nat.Result()
    for name, desc in (("lf_float8_encode", nat.Float8EncodeDesc()), ("lf_float8_decode", nat.Float8DecodeDesc()), ("lf_layer_norm_run", nat.LayerNormDesc()),
                       ("lf_layer_norm_backward_run", nat.LayerNormBackwardDesc()), ("lf_float8_linear_run", nat.Float8LinearDesc()),
                       ("lf_float8_weight_gradient_run", nat.Float8WeightGradientDesc())):
        assert getattr(lib, name)(None, ctypes.byref(desc), res) == nat.LF_ERR_ARGUMENT
    assert lib.lf_layer_norm_backward_workspace(None, 4, 4) == 0 and lib.lf_float8_weight_gradient_workspace(None, 4, 4, 4) == 0
    assert lib.lf_float8_code_bytes(0, 4) == 0 and lib.lf_float8_exponent_bytes(4, -1) == 0 and lib.lf_float8_linear_workspace(-1, 4) == 0
