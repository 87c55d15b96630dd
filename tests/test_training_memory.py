"""Tensors that stand for others - fake, wrapped by a function transform, of a subclass: refused, or without a trace in later calls."""
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import localfold_b200 as lf
from localfold_b200 import training
from test_training_refusals import DEVICE, Fake, float8, weights

NO_MEMORY = "must be a tensor with memory of its own"


@pytest.fixture(autouse=True)
def prototypes(monkeypatch):
    """Nothing of other tests' calls, and nothing left for them."""
    kept = {}
    monkeypatch.setattr(training, "_empty", kept)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")      # (torch warns of a fake tensor's address)
        yield kept


class Unallocated(Fake):
    def data_ptr(self):
        return 0


class Wrapped(Fake):
    def data_ptr(self):
        raise RuntimeError("Cannot access data pointer of Tensor that doesn't have storage")


@pytest.mark.parametrize("kind", [Unallocated, Wrapped])
def test_arguments_without_memory(kind):
    norm, linear = lf.LayerNormGpu(DEVICE), lf.Float8LinearGpu(DEVICE)
    x, of8, of4 = kind(32), Fake(8), Fake(4)
    shape = {"rows": 4, "channels": 8}
    calls = {
        "encode": lambda: lf.float8_encode(DEVICE, x, 4, 8),
        "norm": lambda: norm.run({**shape, "activations": x, "scale": of8, "offset": of8}, {"checkpoint": "e4m3"}),
        "scale": lambda: norm.run({**shape, "activations": Fake(32), "scale": kind(8), "offset": of8}),
        "backward": lambda: norm.backward({**shape, "gradient": x, "activations": Fake(32), "mean": of4, "inverseDeviation": of4, "scale": of8}),
        "product": lambda: linear.run({**shape, "outChannels": 6, "activations": x, "weights": weights(6, 8)}),
        "out": lambda: linear.run({**shape, "outChannels": 6, "activations": float8(4, 8), "weights": weights(6, 8)}, {"output": "f32"}, kind(24)),
        "memory": lambda: lf.Float8Tensor(4, 8, "e4m3", kind(sum(training._sizes(4, 8)), torch.uint8)),
    }
    for call in calls.values():
        with pytest.raises(ValueError, match=NO_MEMORY):
            call()


def test_fake_tensors_leave_nothing_behind(prototypes):
    with FakeTensorMode():
        x, of8 = torch.empty(32, device="cuda"), torch.empty(8, device="cuda")
    assert type(x) is not torch.Tensor and x.is_cuda
    with pytest.raises(ValueError, match=NO_MEMORY):
        lf.float8_encode(DEVICE, x, 4, 8)
    with pytest.raises(ValueError, match=NO_MEMORY):
        lf.LayerNormGpu(DEVICE).run({"rows": 4, "channels": 8, "activations": x, "scale": of8, "offset": of8}, {"checkpoint": "e4m3"})
    assert not prototypes


@pytest.mark.parametrize("real", [False, True])
@pytest.mark.parametrize("dtype", ["bytes", "f32", "bf16"])
def test_memory_under_a_fake_mode(prototypes, dtype, real):
    """No result without memory, neither under the mode nor after it."""
    like = torch.ones(3)
    if real:
        training._new(like, dtype, 4)
    for mode in (FakeTensorMode(), FakeTensorMode(allow_non_fake_inputs=True)):
        with mode, pytest.raises((ValueError, AssertionError)):
            training._new(like, dtype, 4)
    after = training._new(like, dtype, (2, 3))
    assert type(after) is torch.Tensor and after.data_ptr() and after.shape == (2, 3)


class Subclass(torch.Tensor):
    pass


def test_memory_is_plain(prototypes):
    """Whatever the first tensor of a kind was."""
    for like in (torch.ones(3).as_subclass(Subclass), torch.nn.Parameter(torch.ones(3))):
        prototypes.clear()
        for _ in range(2):
            got = training._new(like, "f32", (2, 2))
            assert type(got) is torch.Tensor and not got.requires_grad and got.dtype == torch.float32
    prototypes.clear()
    with torch.inference_mode():
        training._new(torch.ones(3), "f32", 2)
    assert not next(iter(prototypes.values())).is_inference()


def test_function_transforms_leave_nothing_behind(prototypes):
    def f(t):
        training._new(t, "f32", 2).data_ptr()
        return t.sum()

    with pytest.raises(RuntimeError, match="data pointer"):
        torch.func.grad(f)(torch.ones(3))
    assert training._new(torch.ones(3), "f32", 2).data_ptr()


@pytest.mark.gpu
def test_results_are_plain():
    """A subclass with memory of its own is an input like another; results are plain tensors, and later calls' too."""
    d = lf.Device(0)
    x, scale = torch.randn(40, 128, device="cuda"), torch.nn.Parameter(torch.rand(128, device="cuda"))
    results = []
    for given in (x.as_subclass(Subclass), x):
        a = lf.LayerNormGpu(d).run({"rows": 40, "channels": 128, "activations": given, "scale": scale, "offset": scale}, {"checkpoint": "e4m3"})
        back = lf.LayerNormGpu(d).backward({"rows": 40, "channels": 128, "gradient": given, "activations": a["checkpoint"], "mean": a["mean"],
                                            "inverseDeviation": a["inverseDeviation"], "scale": scale})
        results.append([a["output"], a["mean"], lf.float8_decode(d, a["checkpoint"]), back["activations"], back["scale"], back["offset"]])
    d.synchronize()
    for one, two in zip(*results):
        assert type(one) is type(two) is torch.Tensor and not one.requires_grad and torch.equal(one, two)
    d.close()
