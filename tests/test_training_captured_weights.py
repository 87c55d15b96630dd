"""Weights of one device in calls of another that are captured into a graph."""
import pytest
import torch

import fake_cuda
import localfold_b200 as lf
from localfold_b200 import training
from test_training_refusals import Fake, FakeDevice, float8, weights

WAIT = """
stream, other = lib.lf_context_stream(context), 64
fake.fake_capture.argtypes = [ctypes.c_void_p]
assert lib.lf_context_await(context, other) == nat.LF_OK and fake.fake_recorded() == 1
fake.fake_capture(stream)
assert lib.lf_context_await(context, other) == nat.LF_ERR_UNSUPPORTED and fake.fake_recorded() == 1
print(lib.lf_last_error(context).decode())
assert lib.lf_context_await(context, stream) == nat.LF_OK
fake.fake_capture(other)      # (work of this context joins a capture elsewhere)
assert lib.lf_context_await(context, other) == nat.LF_OK and fake.fake_recorded() == 2
"""


def test_wait_in_a_capture_is_refused(tmp_path):
    assert "a call that is being captured cannot wait" in fake_cuda.run(tmp_path, WAIT)


def test_captured_calls_do_not_wait(monkeypatch):
    """A device waits for the weights with every call (their own may replay a graph that encodes them), but for captured ones after the first since an update."""
    capturing = []
    monkeypatch.setattr(training, "_torch_stream", lambda ordinal: 1 if not capturing else capturing[0])
    monkeypatch.setattr(training, "_capturing", lambda: bool(capturing))
    log = []
    owner, users = FakeDevice(log, 1), [FakeDevice(log, 2), FakeDevice(log, 3)]
    w, value = weights(6, 8), Fake(48)
    w.device, value.shape = owner, (6, 8)
    call = {"rows": 4, "channels": 8, "outChannels": 6, "activations": float8(4, 8), "weights": w}
    back = {"rows": 4, "channels": 8, "outChannels": 6, "gradient": float8(4, 6), "weights": w}
    for _ in range(3):
        for user in users:
            log.clear()
            for captured in (False, True, False, True):
                capturing[:] = [user.stream] if captured else []
                lf.Float8LinearGpu(user).run(call, None, Fake(24, torch.bfloat16))
                lf.Float8LinearGpu(user).input_gradient(back, None, Fake(32, torch.bfloat16))
            assert [e[1:3] for e in log if e[0] == "lf_context_await"] == 4 * [(user.stream, 1)]
        capturing.clear()
        log.clear()
        w.update(value)
        assert sorted(e[1:3] for e in log if e[0] == "lf_context_await") == [(1, 2), (1, 3)] and log[-1][0] == "lf_float8_encode"
        log.clear()
        capturing[:] = [2]      # (the first call after an update: the library refuses the wait)
        lf.Float8LinearGpu(users[0]).run(call, None, Fake(24, torch.bfloat16))
        assert [e[1:3] for e in log if e[0] == "lf_context_await"] == [(2, 1)]
        capturing.clear()


def test_update_after_close_is_refused(monkeypatch):
    """The context that would encode the values is gone."""
    monkeypatch.setattr(training, "_torch_stream", lambda ordinal: 1)
    log = []
    owner, w, value = FakeDevice(log, 1), weights(6, 8), Fake(48)
    w.device, value.shape = owner, (6, 8)
    w.update(value)
    owner._finalizer.alive = False
    with pytest.raises(ValueError, match="the weights' device is closed"):
        w.update(value)
    assert [e[0] for e in log] == ["lf_float8_encode"]


@pytest.mark.parametrize("own", [False, True])
def test_capture_on_another_stream_is_refused(monkeypatch, own):
    """... before anything of the call has reached the device's stream."""
    monkeypatch.setattr(training, "_torch_stream", lambda ordinal: 1)
    monkeypatch.setattr(training, "_capturing", lambda: True)
    log = []
    d, w = FakeDevice(log, 2), weights(6, 8)
    d._own_stream, w.device = own, d
    call = {"rows": 4, "channels": 8, "outChannels": 6, "activations": float8(4, 8), "weights": w}
    with pytest.raises(RuntimeError, match="a call is captured on its device's stream"):
        lf.Float8LinearGpu(d).run(call, None, Fake(24, torch.bfloat16))
    assert not log
    d.stream = 1
    lf.Float8LinearGpu(d).run(call, None, Fake(24, torch.bfloat16))
    assert [e[0] for e in log] == ["lf_float8_linear_run"]


@pytest.mark.gpu
def test_capture_goes_on_after_a_refusal():
    """A device with a stream of its own, called while torch captures another: refused, the graph holds the rest, and the device works as before."""
    d = lf.Device(0)
    x = torch.randn(64, 128, device="cuda")
    want = lf.float8_decode(d, lf.float8_encode(d, x, 64, 128), {"output": "f32"})
    d.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        y = x * 2
        with pytest.raises(RuntimeError, match="a call is captured on its device's stream"):
            lf.float8_encode(d, x, 64, 128)
        z = y + 1
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, x * 2 + 1)
    got = lf.float8_decode(d, lf.float8_encode(d, x, 64, 128), {"output": "f32"})
    d.synchronize()
    assert torch.equal(got, want)
    d.close()


@pytest.mark.gpu
def test_captured_on_another_device():
    stream = torch.cuda.Stream()
    owner, user = lf.Device(0), lf.Device(0, stream=stream.cuda_stream)
    x, first, second = torch.randn(300, 512, device="cuda"), torch.randn(400, 512, device="cuda"), torch.randn(400, 512, device="cuda")
    w = lf.prepare_float8_linear_weights(owner, first)
    call = {"rows": 300, "channels": 512, "outChannels": 400, "activations": x, "weights": w}
    owner.synchronize()
    torch.cuda.synchronize()
    linear = lf.Float8LinearGpu(user)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        linear.run({**call, "weights": lf.prepare_float8_linear_weights(user, first)})      # (modules are loaded)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            with pytest.raises(NotImplementedError, match="a call that is being captured cannot wait"):
                linear.run(call)
            x.add_(0)      # (the capture goes on)
        graph = torch.cuda.CUDAGraph()
        want = linear.run(call)["output"]
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            got = linear.run(call)["output"]
        graph.replay()
    stream.synchronize()
    assert torch.equal(got, want)
    w.update(second)
    owner.synchronize()
    with torch.cuda.stream(stream):
        graph.replay()
        new = linear.run(call)["output"]
    stream.synchronize()
    assert torch.equal(got, new) and not torch.equal(got, want)
    owner.close()
    user.close()


@pytest.mark.gpu
def test_weights_that_a_graph_encodes():
    """A graph on the weights' stream encodes them anew at each replay, behind a queue; another device's next call has the new values."""
    n = 2048
    stream = torch.cuda.Stream()
    owner, user = lf.Device(0, stream=stream.cuda_stream), lf.Device(0)
    source, x = torch.zeros(n, n, device="cuda"), torch.randn(64, n, device="cuda")
    w = lf.prepare_float8_linear_weights(owner, source)
    call, linear = {"rows": 64, "channels": n, "outChannels": n, "activations": x, "weights": w}, lf.Float8LinearGpu(user)
    torch.cuda.synchronize()
    a, graph = torch.randn(n, n, device="cuda"), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        w.update(source)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            w.update(source)
    linear.run(call)
    user.synchronize()
    for _ in range(5):
        fresh = torch.randn(n, n, device="cuda")
        want = linear.run({**call, "weights": lf.prepare_float8_linear_weights(user, fresh)})["output"]
        user.synchronize()
        source.copy_(fresh)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(30):
                a = (a @ a) * 1e-2
            graph.replay()
        got = linear.run(call)["output"]
        user.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    owner.close()
    user.close()
