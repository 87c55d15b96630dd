"""The training operators as they are used: one after the other, in CUDA graphs, on streams of their own, on large tensors, and what the library
refuses before a launch."""
import ctypes

import numpy as np
import pytest
import torch

import training_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    import localfold_b200 as lf
    d = lf.Device(0)
    yield d
    d.close()


def host(t):
    return t.double().cpu().numpy()


def problem(seed, rows, c, n, dtype=torch.bfloat16):
    rng = np.random.default_rng(seed)
    x = torch.as_tensor(rng.standard_normal((rows, c)) + 0.5 * rng.standard_normal(c)).to(dtype).cuda()
    g, b = (torch.as_tensor(t).float().cuda() for t in (1 + 0.2 * rng.standard_normal(c), 0.2 * rng.standard_normal(c)))
    w, bias = (torch.as_tensor(t).float().cuda() for t in (rng.standard_normal((n, c)) / np.sqrt(c), 0.1 * rng.standard_normal(n)))
    dy = torch.as_tensor(1e-3 * rng.standard_normal((rows, n))).to(dtype).cuda()
    return x, g, b, w, bias, dy


def step(dev, x, g, b, w, bias, dy, weights=None):
    """A norm and its projection, forward and backward: the 8-bit output of the norm is the projection's operand and its checkpoint."""
    import localfold_b200 as lf
    (rows, c), n = x.shape, w.shape[0]
    norm, linear = lf.LayerNormGpu(dev), lf.Float8LinearGpu(dev)
    if weights is None:
        weights = lf.prepare_float8_linear_weights(dev, w, bias)
    else:
        weights.update(w, bias)
    shape = {"rows": rows, "channels": c, "outChannels": n}
    a = norm.run({"rows": rows, "channels": c, "activations": x, "scale": g, "offset": b}, {"checkpoint": "e4m3", "encode": "e4m3"})
    y = linear.run({**shape, "activations": a["output"], "weights": weights})
    back = linear.input_gradient({**shape, "gradient": dy, "weights": weights}, {"output": "bf16"})
    grads = linear.weight_gradient({**shape, "gradient": dy, "activations": a["output"]})
    d = norm.backward({"rows": rows, "channels": c, "gradient": back["output"], "activations": a["checkpoint"], "mean": a["mean"],
                       "inverseDeviation": a["inverseDeviation"], "scale": g})
    return {"y": y["output"], "weight": grads["weight"], "bias": grads["bias"], "x": d["activations"], "scale": d["scale"], "offset": d["offset"]}


@pytest.mark.parametrize("rows,c,n", [(7, 64, 40), (300, 128, 512), (1025, 384, 200)])
def test_step(dev, rows, c, n):
    """Against 64 bits, with the roundings that the operators declare taken from their own 8-bit values: each operator is compared for itself elsewhere, here what one
    hands to the next.  The norm's 8-bit output may differ from the 64-bit norm's by one code where its float32 value lies next to a border."""
    import localfold_b200 as lf
    x, g, b, w, bias, dy = problem(rows, rows, c, n)
    got = step(dev, x, g, b, w, bias, dy)
    norm = lf.LayerNormGpu(dev).run({"rows": rows, "channels": c, "activations": x, "scale": g, "offset": b}, {"checkpoint": "e4m3", "encode": "e4m3"})
    a8, x8 = (lf.float8_decode(dev, norm[k], {"output": "f32"}) for k in ("output", "checkpoint"))
    dev.synchronize()
    a8, w8, d8 = host(a8), ref.decoded(host(w), "e4m3", 128), ref.decoded(host(dy))
    want, mean, inverse = ref.layer_norm(host(x), host(g), host(b))
    # a code is off by half a step, 2^-4 of the value and 2^-10 of the block's unit (the least code), next to a border by another such half
    unit = np.exp2(ref.exponents(want)).repeat(128, 1)[:, :c]
    ref.close(a8, want, 2 * (2.0 ** -4 * np.abs(want) + 2.0 ** -10 * unit) + 1e-4, "norm in 8 bits")
    y = a8 @ w8.T + host(bias)
    size = np.abs(a8) @ np.abs(w8).T + np.abs(host(bias))
    ref.close(got["y"], y, c * 2.0 ** -23 * size + 2.0 ** -8 * np.abs(y) + 2.0 ** -23 * size, "output")
    da = d8 @ w8
    da_size = np.abs(d8) @ np.abs(w8)
    chain = (rows / 16 + 164) * 2.0 ** -23
    ref.close(got["weight"], host(dy).T @ a8, chain * (np.abs(host(dy)).T @ np.abs(a8)), "weight")
    ref.close(got["bias"], host(dy).sum(0), chain * np.abs(host(dy)).sum(0), "bias")
    # the norm's gradient of a gradient that was rounded to bf16 and may be off by the product's error: linear in it.  Statistics and sums are float32: 128 U, U =
    # 2^-24, times (|x| / deviation)^2 < 10 is below 1e-4.
    off = 2.0 ** -8 * np.abs(da) + n * 2.0 ** -23 * da_size
    dx, dg, db = ref.layer_norm_backward(da, host(x8), mean, inverse, host(g))
    u = np.abs(host(x8) - mean[:, None]) * inverse[:, None]
    h = off * np.abs(host(g))
    spread = inverse[:, None] * (h + h.mean(1, keepdims=True) + u * (h * u).mean(1, keepdims=True))
    ref.close(got["x"], dx, 1.01 * spread + 2.0 ** -8 * np.abs(dx) + 1e-4 * np.abs(dx).max(), "input")
    ref.close(got["scale"], dg, 1.01 * (off * u).sum(0) + 1e-5 * (np.abs(da) * u).sum(0), "scale")
    ref.close(got["offset"], db, 1.01 * off.sum(0) + 1e-5 * np.abs(da).sum(0), "offset")


def test_gradient_follows_the_loss(dev):
    """The weight's gradient against differences of the forward pass: the product is linear in the weight's 8-bit values, so moving by whole codes is exact."""
    import localfold_b200 as lf
    x, _, _, _, _, dy = problem(3, 96, 128, 24)
    w = torch.zeros(24, 128, device="cuda")
    w[:, 0] = 1.0      # the blocks' unit stays what this value makes it
    linear = lf.Float8LinearGpu(dev)
    shape = {"rows": 96, "channels": 128, "outChannels": 24}
    x8 = lf.float8_encode(dev, x, 96, 128)
    grads = linear.weight_gradient({**shape, "gradient": dy, "activations": x8})

    def loss(weight):
        y = linear.run({**shape, "activations": x8, "weights": lf.prepare_float8_linear_weights(dev, weight)}, {"output": "f32"})["output"]
        dev.synchronize()
        return (host(y) * host(dy)).sum()

    for n, k in ((0, 1), (5, 77), (23, 127)):
        up, down = w.clone(), w.clone()
        up[n, k], down[n, k] = 0.5, -0.5
        difference = loss(up) - loss(down)
        dev.synchronize()
        scale = float(np.abs(host(dy)[:, n] * 8).sum())
        assert abs(float(grads["weight"][n, k]) - difference) <= 128 * 2.0 ** -23 * scale


def test_one_stream_and_another(dev):
    """A device on torch's stream, one with a stream of its own, one on a side stream: the same bits."""
    import localfold_b200 as lf
    args = problem(11, 500, 200, 72)
    want = step(dev, *args)
    dev.synchronize()
    ours = lf.Device(0, stream=torch.cuda.current_stream().cuda_stream)
    got = step(ours, *args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    other = lf.Device(0, stream=side.cuda_stream)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = step(other, *args)
    side.synchronize()
    fourth = step(other, *args)      # torch's current stream is not the device's now: inputs are ready, memory is kept for that stream
    side.synchronize()
    for name, value in want.items():
        for result in (got, third, fourth):
            assert torch.equal(result[name], value), name
    ours.close()
    other.close()


def test_weights_of_another_device(dev):
    """Weights encoded on one device's stream and used on another's: the second waits for them."""
    import localfold_b200 as lf
    other = lf.Device(0)
    x = torch.randn(64, 2048, device="cuda")
    shape = {"rows": 64, "channels": 2048, "outChannels": 4096}
    first = torch.randn(4096, 2048, device="cuda")
    weights = lf.prepare_float8_linear_weights(other, first)
    other.synchronize()
    for _ in range(10):
        w = torch.randn(4096, 2048, device="cuda")
        weights.update(w)
        got = lf.Float8LinearGpu(dev).run({**shape, "activations": x, "weights": weights})["output"]
        dev.synchronize()
        want = lf.Float8LinearGpu(other).run({**shape, "activations": x, "weights": weights})["output"]
        other.synchronize()
        assert torch.equal(got, want)
    other.close()


def test_memory_is_not_reused_too_early():
    """A device with a stream of its own: results dropped at once, their memory used again by torch while the calls may still run."""
    import localfold_b200 as lf
    d = lf.Device(0)
    x = torch.randn(200000, 128, device="cuda")
    want = lf.float8_decode(d, lf.float8_encode(d, x, 200000, 128), {"output": "f32"})
    d.synchronize()
    for _ in range(20):
        got = lf.float8_decode(d, lf.float8_encode(d, x, 200000, 128), {"output": "f32"})      # (the encoded matrix is dropped before it is read)
        junk = torch.full((30_000_000,), 255, dtype=torch.uint8, device="cuda")
        del junk
    d.synchronize()
    assert torch.equal(got, want)
    d.close()


def test_captured(dev):
    """Two graphs of the step, replayed in turn with new inputs, beside eager calls: each has results of its own."""
    import localfold_b200 as lf
    stream = torch.cuda.Stream()
    d = lf.Device(0, stream=stream.cuda_stream)
    cases = [problem(21, 400, 128, 256), problem(22, 150, 264, 72)]
    graphs = []
    with torch.cuda.stream(stream):
        for args in cases:
            weights = lf.prepare_float8_linear_weights(d, args[3], args[4])
            step(d, *args, weights)      # a first call outside: modules load at the first launch
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                results = step(d, *args, weights)
            graphs.append((graph, results, weights))      # (what a graph reads and writes lives as long as it)
    for turn in range(3):
        for args, (graph, results, _) in zip(cases, graphs):
            fresh = problem(100 + turn, args[0].shape[0], args[0].shape[1], args[3].shape[0])
            for old, new in zip(args, fresh):
                old.copy_(new)
            torch.cuda.synchronize()
            graph.replay()
            with torch.cuda.stream(stream):
                step(d, *problem(7, 90, 96, 40))      # eager work between the replays
            torch.cuda.synchronize()
            want = step(dev, *fresh)
            dev.synchronize()
            for name, value in want.items():
                assert torch.equal(results[name], value), (turn, name)
    d.close()


def test_replayed_at_the_same_time(dev):
    """Graphs of one device's calls have workspaces of their own: replayed on two streams at once they do not meet."""
    import localfold_b200 as lf
    stream = torch.cuda.Stream()
    d = lf.Device(0, stream=stream.cuda_stream)
    cases = [problem(31, 3000, 128, 512), problem(32, 2500, 512, 128)]
    graphs = []
    with torch.cuda.stream(stream):
        for args in cases:
            weights = lf.prepare_float8_linear_weights(d, args[3], args[4])
            step(d, *args, weights)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                results = step(d, *args, weights)
            graphs.append((graph, results, weights))      # (what a graph reads and writes lives as long as it)
    wants = [step(dev, *args) for args in cases]
    dev.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for s, (graph, *_) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for want, (_, results, _) in zip(wants, graphs):
        for name, value in want.items():
            assert torch.equal(results[name], value), name
    d.close()


def test_past_32_bits(dev):
    """More than 2^32 bytes and 2^31 elements: the last rows are where they belong (compared with calls on those rows alone)."""
    import localfold_b200 as lf
    rows, c, last = 17_000_003, 128, 1000
    x = torch.empty(rows, c, dtype=torch.bfloat16, device="cuda")
    x.normal_()
    tail = x[-last:].clone()
    g, b = torch.rand(c, device="cuda") + 0.5, torch.randn(c, device="cuda")
    norm = lf.LayerNormGpu(dev)
    a = norm.run({"rows": rows, "channels": c, "activations": x, "scale": g, "offset": b}, {"checkpoint": "e4m3"})
    t = norm.run({"rows": last, "channels": c, "activations": tail, "scale": g, "offset": b}, {"checkpoint": "e4m3"})
    dev.synchronize()
    assert torch.equal(a["output"][-last:], t["output"]) and torch.equal(a["mean"][-last:], t["mean"])
    values = lf.float8_decode(dev, a["checkpoint"])
    want = lf.float8_decode(dev, t["checkpoint"])
    dev.synchronize()
    assert torch.equal(values[-last:], want)
    back = norm.backward({"rows": rows, "channels": c, "gradient": x, "activations": a["checkpoint"], "mean": a["mean"],
                          "inverseDeviation": a["inverseDeviation"], "scale": g}, out=values)
    part = norm.backward({"rows": last, "channels": c, "gradient": tail, "activations": t["checkpoint"], "mean": t["mean"],
                          "inverseDeviation": t["inverseDeviation"], "scale": g})
    dev.synchronize()
    assert torch.equal(back["activations"][-last:], part["activations"])
    linear, weights = lf.Float8LinearGpu(dev), lf.prepare_float8_linear_weights(dev, torch.randn(160, c, device="cuda"))
    y = linear.run({"rows": rows, "channels": c, "outChannels": 160, "activations": a["checkpoint"], "weights": weights})
    z = linear.run({"rows": last, "channels": c, "outChannels": 160, "activations": t["checkpoint"], "weights": weights})
    dev.synchronize()
    assert torch.equal(y["output"][-last:], z["output"])


@pytest.mark.parametrize("rows,c,n,dtype", [(37, 72, 40, torch.bfloat16), (130, 33, 77, torch.float32), (3, 50, 9, torch.bfloat16), (700, 128, 256, torch.float32)])
def test_nothing_behind_the_last_row(dev, rows, c, n, dtype):
    """Outputs in the middle of larger memory, at addresses that no 16-byte access divides too: what surrounds them stays."""
    import localfold_b200 as lf
    x, g, b, w, bias, dy = problem(rows, rows, c, n, dtype)
    weights = lf.prepare_float8_linear_weights(dev, w, bias)
    shape = {"rows": rows, "channels": c, "outChannels": n, "weights": weights}
    for shift in (0, 1, 8):
        def room(count):
            t = torch.full((count + 64,), 3.0, dtype=dtype, device="cuda")
            return t, t[shift:shift + count]
        (y_all, y), (z_all, z) = room(rows * n), room(rows * c)
        lf.Float8LinearGpu(dev).run({**shape, "activations": x}, None, y.view(rows, n))
        lf.LayerNormGpu(dev).run({"rows": rows, "channels": c, "activations": x, "scale": g, "offset": b}, None, z.view(rows, c))
        plain = lf.Float8LinearGpu(dev).run({**shape, "activations": x})["output"]
        dev.synchronize()
        assert torch.equal(y.view(rows, n), plain)
        for whole, count in ((y_all, rows * n), (z_all, rows * c)):
            assert (whole[:shift] == 3).all() and (whole[shift + count:] == 3).all()


def test_bundle_weights(dev):
    """A weight as a bundle stores it (int5) is decoded, then encoded."""
    import localfold_b200 as lf
    from bundle_writer import int5_payload
    weight = np.random.default_rng(4).standard_normal((96, 64)).astype(np.float32)
    payload, scale_offset, zero_offset = int5_payload(weight)
    encoded = lf.EncodedTensor(payload, scale_offset, zero_offset, weight.size, weight.shape)
    weights = lf.prepare_float8_linear_weights(dev, encoded)
    got = lf.float8_decode(dev, weights.forward, {"output": "f32"})
    dev.synchronize()
    ref.close(got, ref.decoded(encoded.decode(), "e4m3", 128), 0.0)


def test_library_refusals(dev):
    """Descriptors that the library answers with a status and a message, before anything is launched."""
    import localfold_b200 as lf
    from localfold_b200 import _native as nat
    x = torch.zeros(64, 64, device="cuda")
    x8 = lf.float8_encode(dev, x, 64, 64)
    w8 = lf.prepare_float8_linear_weights(dev, x).forward
    out = torch.zeros(64, 64, device="cuda")
    p, ones = x.data_ptr(), torch.ones(64, device="cuda").data_ptr()
    M = lambda t=x8, **k: nat.Float8Matrix(**{**dict(zip(("rows", "channels", "format", "codes", "exponents"), t.fields)), **k})      # noqa: E731
    none = nat.Float8Matrix()
    dev.synchronize()
    launched = dev.launch_count()

    def refuse(function, desc, status, text):
        res = nat.Result()
        assert getattr(dev.lib, function)(dev.handle, ctypes.byref(desc), res) == status
        assert text in dev.lib.lf_last_error(dev.handle).decode()

    A, S, U = nat.LF_ERR_ARGUMENT, nat.LF_ERR_SHAPE, nat.LF_ERR_UNSUPPORTED
    odd = x8.fields[3] + 4
    refuse("lf_float8_encode", nat.Float8EncodeDesc(M(), none, 0, 1, None), A, "null argument")
    refuse("lf_float8_encode", nat.Float8EncodeDesc(M(codes=odd), none, 0, 1, p), A, "16-byte boundaries")
    refuse("lf_float8_encode", nat.Float8EncodeDesc(M(rows=0), none, 0, 1, p), S, "positive")
    refuse("lf_float8_encode", nat.Float8EncodeDesc(M(rows=1 << 31), none, 0, 1, p), U, "too many")
    refuse("lf_float8_encode", nat.Float8EncodeDesc(M(format=2), none, 0, 1, p), A, "format")
    refuse("lf_float8_encode", nat.Float8EncodeDesc(M(), none, 3, 1, p), A, "dtype")
    refuse("lf_float8_encode", nat.Float8EncodeDesc(M(), none, 0, 64, p), A, "1 or 128 rows")
    refuse("lf_float8_encode", nat.Float8EncodeDesc(M(), M(), 0, 1, p), A, "transposed")
    refuse("lf_float8_encode", nat.Float8EncodeDesc(M(rows=63), M(), 0, 128, p), S, "expected 64 x 63")
    refuse("lf_float8_decode", nat.Float8DecodeDesc(M(exponents=None), 0, 0, p), A, "null")
    refuse("lf_float8_decode", nat.Float8DecodeDesc(M(), 0, 0, None), A, "null argument")
    norm = lambda **k: nat.LayerNormDesc(**{**dict(rows=64, channels=64, variance=1, act_dtype=0, epsilon=1e-5, activations=p, scale=ones, offset=ones,      # noqa: E731
                                                   out=out.data_ptr()), **k})
    refuse("lf_layer_norm_run", norm(scale=None), A, "null argument")
    refuse("lf_layer_norm_run", norm(out=None), A, "neither an output")
    refuse("lf_layer_norm_run", norm(mean=ones), A, "come together")
    refuse("lf_layer_norm_run", norm(channels=8193), U, "at most 8192")
    refuse("lf_layer_norm_run", norm(variance=0), A, "variance")
    refuse("lf_layer_norm_run", norm(epsilon=-1.0), S, "epsilon")
    refuse("lf_layer_norm_run", norm(checkpoint=M(channels=65)), S, "expected 64 x 64")
    back = lambda **k: nat.LayerNormBackwardDesc(**{**dict(rows=64, channels=64, act_dtype=0, gradient=p, activations=p, mean=ones, inverse_deviation=ones,      # noqa: E731
                                                           scale=ones, out=out.data_ptr(), scale_gradient=ones, offset_gradient=ones, workspace=p,
                                                           workspace_bytes=x.numel() * 4), **k})
    refuse("lf_layer_norm_backward_run", back(activations=None), A, "null argument")
    refuse("lf_layer_norm_backward_run", back(checkpoint=M()), A, "not both")
    many = dict(rows=4096, channels=1)      # (more rows than one block takes; refused before any of them is read)
    refuse("lf_layer_norm_backward_run", back(**many, workspace_bytes=16), A, "workspace")
    refuse("lf_layer_norm_backward_run", back(**many, workspace=p + 4), A, "workspace")
    lin = lambda **k: nat.Float8LinearDesc(**{**dict(activations=M(), weights=M(w8), out_dtype=0, out=out.data_ptr()), **k})      # noqa: E731
    refuse("lf_float8_linear_run", lin(out=None), A, "null argument")
    refuse("lf_float8_linear_run", lin(weights=M(w8, channels=63)), S, "expected 64 x 64")
    refuse("lf_float8_linear_run", lin(weights=M(w8, format=1)), U, "weights are e4m3")
    refuse("lf_float8_linear_run", lin(activations=M(codes=None)), A, "null")
    refuse("lf_float8_linear_run", lin(activations=M(codes=None), source=p), A, "workspace")
    refuse("lf_float8_linear_run", lin(activations=M(codes=None), source=p, source_dtype=9), A, "source dtype")
    refuse("lf_float8_linear_run", lin(out_dtype=7), A, "dtype")
    grad = lambda **k: nat.Float8WeightGradientDesc(**{**dict(activations=M(), gradient=p, out_channels=64, weight_gradient=out.data_ptr()), **k})      # noqa: E731
    refuse("lf_float8_weight_gradient_run", grad(gradient=None), A, "null argument")
    refuse("lf_float8_weight_gradient_run", grad(encoded_gradient=M()), A, "not both")
    refuse("lf_float8_weight_gradient_run", grad(out_channels=0), S, "positive")
    big = lf.float8_encode(dev, torch.zeros(4096, 64, device="cuda"), 4096, 64)
    launched += 1
    refuse("lf_float8_weight_gradient_run", grad(activations=M(big)), A, "workspace")
    dev.synchronize()
    assert dev.launch_count() == launched and not out.any()


def test_update_while_another_device_reads(dev):
    """Weights of one device, multiplied on another's stream behind a queue of products, and updated at once: the products have the old values."""
    import localfold_b200 as lf
    n = 2048
    x, first, second = (torch.randn(n, n, device="cuda") for _ in range(3))
    weights, other = lf.prepare_float8_linear_weights(dev, first), lf.Device(0)
    dev.synchronize()
    linear, call = lf.Float8LinearGpu(other), {"rows": n, "channels": n, "outChannels": n, "activations": x, "weights": weights}
    want = linear.run(call)["output"]
    other.synchronize()
    got = [linear.run(call)["output"] for _ in range(40)]
    weights.update(second)
    new = linear.run(call)["output"]
    other.synchronize()
    assert all(torch.equal(t, want) for t in got) and not torch.equal(new, want)
    renewed = lf.Float8LinearGpu(dev).run(call)["output"]
    dev.synchronize()
    assert torch.equal(new, renewed)
    other.close()
    weights.update(first)
    again = lf.Float8LinearGpu(dev).run(call)["output"]
    dev.synchronize()
    assert torch.equal(again, want)
