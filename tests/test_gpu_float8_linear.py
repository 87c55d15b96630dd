"""The projection on 8-bit operands and its gradients against 64 bits.

Products of two codes and their powers of two are exact in float32, and so are values of 8-bit forms in bf16; what is off is the sum.  A float32 sum of K
terms is off by at most K 2^-23 sum|terms| to first order (2^-23: additions may truncate), however they are grouped; the
weight's gradient adds products in sixteens (one instruction) and splits, whose chain is rows / 16 and at most 148 splits."""
import numpy as np
import pytest
import torch

import training_reference as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
STEP = 2.0 ** -23
# rows, channels, outputs: single tokens, partial tiles, all tile widths (64, 128, 256 columns), several groups of 512 channels, odd everything
SHAPES = [(1, 1, 1), (1, 16, 8), (3, 128, 64), (4, 1536, 384), (16, 384, 1536), (17, 130, 72), (33, 5, 500), (64, 640, 24), (127, 129, 65), (128, 128, 128), (129, 512, 257),
          (200, 513, 100), (300, 1030, 333), (1000, 64, 1), (2500, 128, 512), (5000, 256, 1000), (20001, 72, 136), (4099, 1200, 640), (30000, 500, 130), (9, 4096, 40), (16, 2000, 33), (8, 5000, 16), (8000, 1100, 1001)]


@pytest.fixture(scope="module")
def dev():
    import localfold_b200 as lf
    d = lf.Device(0)
    yield d
    d.close()


def host(t):
    return t.double().cpu().numpy()


def operands(seed, rows, c, n, dtype):
    """Blocks of very different size, so that a scale taken from the wrong block shows."""
    rng = np.random.default_rng(seed)
    blocks = -(-c // 128)
    x = rng.standard_normal((rows, c)) * np.exp2(rng.integers(-6, 6, (rows, blocks))).repeat(128, 1)[:, :c]
    w = rng.standard_normal((n, c)) * np.exp2(rng.integers(-5, 5, (-(-n // 128), blocks))).repeat(128, 0)[:n].repeat(128, 1)[:, :c]
    dy = rng.standard_normal((rows, n)) * np.exp2(rng.integers(-6, 6, (rows, 1))) * 1e-3
    dy[rows - rows // 20:] = 0
    bias = rng.standard_normal(n)
    return [torch.as_tensor(t).to(TYPES[dtype]).cuda() for t in (x, w, dy)] + [torch.as_tensor(bias).float().cuda()]


@pytest.mark.parametrize("name,dtype", [("e4m3", "f32"), ("e4m3", "bf16"), ("e5m2", "f32"), ("e5m2", "bf16")])
@pytest.mark.parametrize("rows,c,n", SHAPES)
def test_product(dev, rows, c, n, name, dtype):
    import localfold_b200 as lf
    x, w, _, bias = operands(rows + c + n, rows, c, n, dtype)
    weights = lf.prepare_float8_linear_weights(dev, w, bias)
    shape = {"rows": rows, "channels": c, "outChannels": n, "weights": weights}
    linear = lf.Float8LinearGpu(dev)
    got = linear.run({**shape, "activations": x}, {"format": name, "checkpoint": True})
    plain = linear.run({**shape, "activations": x}, {"format": name})
    kept, encoded = (lf.float8_decode(dev, t, {"output": "f32"}) for t in (got["checkpoint"], lf.float8_encode(dev, x, rows, c, {"format": name})))
    weights.bias = None
    again = linear.run({**shape, "activations": got["checkpoint"]}, {"output": "f32"})
    dev.synchronize()
    assert got["output"].dtype == TYPES[dtype] and again["output"].dtype == torch.float32
    assert torch.equal(got["output"], plain["output"]) and "checkpoint" not in plain and torch.equal(kept, encoded)
    x8, w8 = ref.decoded(host(x), name), ref.decoded(host(w), "e4m3", 128)
    want, size = x8 @ w8.T, np.abs(x8) @ np.abs(w8).T
    ref.close(again["output"], want, c * STEP * size, "without a bias, float32")
    want = want + host(bias)
    ref.close(got["output"], want, c * STEP * size + (STEP + ref.half_step(dtype)) * (np.abs(want) + c * STEP * size), dtype)


@pytest.mark.parametrize("name,dtype", [("e4m3", "bf16"), ("e5m2", "f32")])
@pytest.mark.parametrize("rows,c,n", SHAPES)
def test_gradients(dev, rows, c, n, name, dtype):
    import localfold_b200 as lf
    x, w, dy, bias = operands(rows + c + n, rows, c, n, dtype)
    linear, weights = lf.Float8LinearGpu(dev), lf.prepare_float8_linear_weights(dev, w, bias)
    shape = {"rows": rows, "channels": c, "outChannels": n}
    x8 = lf.float8_encode(dev, x, rows, c)
    dx = linear.input_gradient({**shape, "gradient": dy, "weights": weights}, {"format": name, "checkpoint": True, "output": "f32"})
    operand = dx["checkpoint"] if dtype == "f32" else dy
    grads = linear.weight_gradient({**shape, "gradient": operand, "activations": x8})
    same = linear.weight_gradient({**shape, "gradient": operand, "activations": x8})
    dev.synchronize()
    assert torch.equal(grads["weight"], same["weight"]) and torch.equal(grads["bias"], same["bias"])
    xv, wv, dyv = ref.decoded(host(x), "e4m3"), ref.decoded(host(w), "e4m3", 128), ref.decoded(host(dy), name)
    ref.close(dx["output"], dyv @ wv, n * STEP * (np.abs(dyv) @ np.abs(wv)), "input")
    dv = dyv if dtype == "f32" else host(dy)
    chain = (min(rows, 4096) / 16 + 16 + max(rows / 4096, 148)) * STEP
    ref.close(grads["weight"], dv.T @ xv, chain * (np.abs(dv).T @ np.abs(xv)), "weight")
    ref.close(grads["bias"], dv.sum(0), chain * np.abs(dv).sum(0), "bias")


@pytest.mark.parametrize("rows,c,n", [(2048, 4096, 4096), (4000, 4000, 4096), (1500, 2500, 2001), (5000, 1024, 2048), (1999, 1155, 1537), (12001, 2048, 400), (9000, 1000, 333),
                                      (4096, 2048, 1024), (20000, 640, 640), (40000, 1536, 384), (700, 2048, 3000)])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_many_channels(dev, rows, c, n, out):
    """Products of every form of the kernel, pairs of multiprocessors among them; the references are 64-bit products of the decoded operands."""
    import localfold_b200 as lf
    x, w, _, bias = operands(rows + c + n, rows, c, n, "bf16")
    linear, weights = lf.Float8LinearGpu(dev), lf.prepare_float8_linear_weights(dev, w, bias)
    x8 = lf.float8_encode(dev, x, rows, c, {"format": "e5m2" if rows % 2 else "e4m3"})
    call = {"rows": rows, "channels": c, "outChannels": n, "activations": x8, "weights": weights}
    room = torch.full((rows * n + 64,), 7.0, dtype=TYPES[out], device="cuda")
    got, same = linear.run(call, {"output": out}, out=room[:rows * n].view(rows, n))["output"], linear.run(call, {"output": out})["output"]
    a, b = lf.float8_decode(dev, x8, {"output": "f32"}), lf.float8_decode(dev, weights.forward, {"output": "f32"})
    dev.synchronize()
    assert torch.equal(got, same) and (room[rows * n:] == 7).all()
    size, want = a.double().abs() @ b.double().abs().T, a.double() @ b.double().T + bias.double()
    off = c * STEP * size
    bound = off + (STEP + ref.half_step(out)) * (want.abs() + off)
    assert ((got.double() - want).abs() <= bound).all()


def test_forms_at_the_same_time():
    """Captured and replayed, and beside products of other forms on another stream: every form has all of a multiprocessor's tensor memory to itself."""
    import localfold_b200 as lf
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    runs = []
    for stream, sizes in ((first, [(3000, 2048, 2048), (2000, 4096, 4000), (3000, 300, 500)]), (second, [(2500, 2048, 384), (700, 256, 200), (4000, 128, 512)])):
        with torch.cuda.stream(stream):
            device = lf.Device(0, stream=stream.cuda_stream)
            linear, calls = lf.Float8LinearGpu(device), []
            for rows, c, n in sizes:
                weights = lf.prepare_float8_linear_weights(device, torch.randn(n, c, device="cuda"))
                calls.append({"rows": rows, "channels": c, "outChannels": n, "activations": torch.randn(rows, c, device="cuda"), "weights": weights})
            want = [linear.run(call)["output"] for call in calls]
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                got = [linear.run(call)["output"] for call in calls for _ in range(2)]
            runs.append((stream, device, graph, want, got, calls))      # (a graph reads its inputs where they were: they live as long)
    for _ in range(20):
        for stream, _, graph, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, device, _, want, got, _ in runs:
        assert all(torch.equal(got[2 * i], want[i]) and torch.equal(got[2 * i + 1], want[i]) for i in range(len(want)))
        device.synchronize()


@pytest.mark.parametrize("power", [115, -115])
@pytest.mark.parametrize("rows,c,n", [(3, 128, 64), (16, 384, 160), (200, 513, 100), (300, 1030, 700), (300, 4100, 700)])
def test_powers_that_cancel(dev, rows, c, n, power):
    """Activations near one end of float32's range and weights near the other: the products are ordinary numbers, and neither power of two alone
    may take a sum out of the range.  (Powers of two are exact: the bounds are those of ordinary operands.)"""
    import localfold_b200 as lf
    x, w, dy, _ = operands(rows + c + n, rows, c, n, "f32")
    x, w = x * 2.0 ** power, w * 2.0 ** -power
    linear, weights = lf.Float8LinearGpu(dev), lf.prepare_float8_linear_weights(dev, w)
    shape = {"rows": rows, "channels": c, "outChannels": n, "weights": weights}
    y = linear.run({**shape, "activations": x})
    dx = linear.input_gradient({**shape, "gradient": dy * 2.0 ** power})
    dev.synchronize()
    x8, w8, dy8 = ref.decoded(host(x)), ref.decoded(host(w), "e4m3", 128), ref.decoded(host(dy * 2.0 ** power))
    ref.close(y["output"], x8 @ w8.T, c * STEP * (np.abs(x8) @ np.abs(w8).T), "output")
    ref.close(dx["output"], dy8 @ w8, n * STEP * (np.abs(dy8) @ np.abs(w8)), "gradient")


@pytest.mark.parametrize("rows,c,n", [(1, 16, 1), (5, 40, 3), (64, 128, 17), (65, 100, 131), (300, 300, 77), (9000, 128, 2001)])
def test_gradient_at_any_address(dev, rows, c, n):
    """A bf16 gradient that starts at any element, with numbers that are none in front of it and behind: the same bits as from memory of its own."""
    import localfold_b200 as lf
    x8 = lf.float8_encode(dev, torch.randn(rows, c, device="cuda"), rows, c)
    dy = torch.randn(rows, n, device="cuda").bfloat16()
    linear, call = lf.Float8LinearGpu(dev), {"rows": rows, "channels": c, "outChannels": n, "activations": x8}
    want = linear.weight_gradient({**call, "gradient": dy})
    for shift in range(1, 9):
        room = torch.full((rows * n + 32,), float("nan"), dtype=torch.bfloat16, device="cuda")
        view = room[shift:shift + rows * n].view(rows, n)
        view.copy_(dy)
        got = linear.weight_gradient({**call, "gradient": view})
        dev.synchronize()
        assert torch.equal(got["weight"], want["weight"]) and torch.equal(got["bias"], want["bias"]), shift
    values = lf.float8_decode(dev, x8, {"output": "f32"})
    dev.synchronize()
    chain = (min(rows, 4096) / 16 + 16 + max(rows / 4096, 148)) * STEP
    ref.close(want["weight"], host(dy).T @ host(values), chain * (np.abs(host(dy)).T @ np.abs(host(values))), "weight")


def test_long_sums(dev):
    """Values of one sign over many rows, several chains a tile: the bound of a chain holds, and what the tests' shorter sums allow."""
    import localfold_b200 as lf
    rows, c, n = 40000, 300, 1200
    x = torch.rand(rows, c, device="cuda") + 0.5
    dy = (torch.rand(rows, n, device="cuda") + 0.5).bfloat16()
    x8 = lf.float8_encode(dev, x, rows, c)
    values = lf.float8_decode(dev, x8, {"output": "f32"})
    got = lf.Float8LinearGpu(dev).weight_gradient({"rows": rows, "channels": c, "outChannels": n, "gradient": dy, "activations": x8})
    dev.synchronize()
    want = (dy.double().T @ values.double()).cpu().numpy()
    ref.close(got["weight"], want, (4096 / 16 + 16 + 148) * STEP * want, "weight")
    sums = dy.double().sum(0).cpu().numpy()
    ref.close(got["bias"], sums, (4096 / 16 + 16 + 148) * STEP * sums, "bias")
