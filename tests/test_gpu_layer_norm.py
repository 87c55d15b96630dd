"""LayerNorm and its gradients, whole and through the 8-bit checkpoint, against 64 bits.

Bounds: a float32 sum of n terms whose longest chain of additions is d is off by at most d U sum|terms| to first order, U = 2^-24.  A lane adds 8 to 32
terms, a row's tree has 5 to 13 levels more; the mean and the variance each cost one such sum, so 128 U covers a chain of any width here with
room for the handful of multiplications.  An error of the mean moves every element by rstd times it, relative to the row's largest magnitude."""
import numpy as np
import pytest
import torch

import training_reference as ref

pytestmark = pytest.mark.gpu
U = 128 * ref.U32
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# widths: one channel, narrow, one vector, whole blocks, odd, each form's last width and the next one's first
SHAPES = [(1, 1), (3, 5), (129, 8), (1, 128), (65, 64), (300, 65), (77, 100), (64, 128), (1000, 128), (33, 129), (50, 256), (41, 257), (17, 384), (21, 512),
          (9, 513), (13, 1000), (5, 1024), (6, 1025), (3, 2048), (2, 2049), (3, 4096), (2, 4097), (1, 8192), (7, 8191), (40000, 16), (20011, 72), (256, 60), (257, 60), (32, 512), (33, 500)]      # (the last four: one block and two)


@pytest.fixture(scope="module")
def dev():
    import localfold_b200 as lf
    d = lf.Device(0)
    yield d
    d.close()


def tensors(seed, rows, c, dtype, spread=2.0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, c)) * np.exp(0.5 * rng.standard_normal((rows, 1))) + spread * rng.standard_normal(c)
    g, b = 1 + 0.3 * rng.standard_normal(c), 0.3 * rng.standard_normal(c)
    x = torch.as_tensor(x).to(TYPES[dtype]).cuda()
    return x, torch.as_tensor(g).float().cuda(), torch.as_tensor(b).float().cuda(), rng


def host(t):
    return t.double().cpu().numpy()


def forward_bounds(x, want, inverse, scale, dtype):
    most = np.abs(x).max(1, keepdims=True)
    return U * (most * inverse[:, None] * np.abs(scale) * (1 + (most * inverse[:, None])) + np.abs(want) + 1) + ref.half_step(dtype) * np.abs(want)


def run(dev, x, g, b, options=None, **more):
    import localfold_b200 as lf
    rows, c = x.shape
    return lf.LayerNormGpu(dev).run({"rows": rows, "channels": c, "activations": x, "scale": g, "offset": b, **more}, options)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,c", SHAPES)
def test_forward(dev, rows, c, dtype):
    x, g, b, _ = tensors(rows * 10007 + c, rows, c, dtype)
    got = run(dev, x, g, b, {"statistics": True})
    dev.synchronize()
    want, mean, inverse = ref.layer_norm(host(x), host(g), host(b))
    ref.close(got["output"], want, forward_bounds(host(x), want, inverse, host(g), dtype), "output")
    most = np.abs(host(x)).max(1)
    ref.close(got["mean"], mean, U * most, "mean")
    ref.close(got["inverseDeviation"], inverse, U * inverse * (1 + (most * inverse) ** 2), "inverse deviation")
    assert got["launches"] == 1 and "checkpoint" not in got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,c", SHAPES)
@pytest.mark.parametrize("kept", ["", "e4m3", "e5m2"])
def test_gradients(dev, rows, c, dtype, kept):
    """From the statistics that the forward pass left; the checkpoint's values are the input then."""
    import localfold_b200 as lf
    x, g, b, rng = tensors(rows * 10007 + c, rows, c, dtype)
    dy = torch.as_tensor(rng.standard_normal((rows, c)) * 1e-2).to(TYPES[dtype]).cuda()
    dy[rows - rows // 20:] = 0
    forward = run(dev, x, g, b, {"checkpoint": kept} if kept else {"statistics": True})
    got = lf.LayerNormGpu(dev).backward({"rows": rows, "channels": c, "gradient": dy, "activations": forward["checkpoint"] if kept else x,
                                         "mean": forward["mean"], "inverseDeviation": forward["inverseDeviation"], "scale": g})
    dev.synchronize()
    if kept:
        values = ref.decoded(host(x), kept)
        decoded = lf.float8_decode(dev, forward["checkpoint"], {"output": "f32"})
        dev.synchronize()
        ref.close(decoded, values, 0.0, "checkpoint")
    else:
        values = host(x)
    mean, inverse = host(forward["mean"]), host(forward["inverseDeviation"])
    dx, dg, db = ref.layer_norm_backward(host(dy), values, mean, inverse, host(g))
    u = np.abs(values - mean[:, None]) * inverse[:, None] + np.abs(mean)[:, None] * inverse[:, None]      # (the difference is rounded as it is taken)
    h = np.abs(host(dy) * host(g))
    size = inverse[:, None] * (h + h.mean(1, keepdims=True) + u * (h * u).mean(1, keepdims=True))
    ref.close(got["activations"], dx, U * size + ref.half_step(dtype) * np.abs(dx), "activations")
    # rows add up in lanes (at most rows / blocks of them in a chain), groups, blocks and strands: fewer than 256 steps at these sizes
    ref.close(got["scale"], dg, 2 * U * (np.abs(host(dy)) * u).sum(0), "scale")
    ref.close(got["offset"], db, 2 * U * np.abs(host(dy)).sum(0), "offset")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("c", [3, 8, 40, 128, 200, 1030])
def test_differences(dev, c, dtype):
    """The input's gradient against central differences of the 64-bit forward pass along a direction: d = sum(dy (y(x + t v) - y(x - t v))) / 2t."""
    import localfold_b200 as lf
    rows = 4
    x, g, b, rng = tensors(c, rows, c, dtype)
    dy = torch.as_tensor(rng.standard_normal((rows, c))).to(TYPES[dtype]).cuda()
    forward = run(dev, x, g, b, {"statistics": True})
    got = lf.LayerNormGpu(dev).backward({"rows": rows, "channels": c, "gradient": dy, "activations": x, "mean": forward["mean"],
                                         "inverseDeviation": forward["inverseDeviation"], "scale": g})
    dev.synchronize()
    v, t = rng.standard_normal((rows, c)), 1e-5
    y = [ref.layer_norm(host(x) + s * t * v, host(g), host(b))[0] for s in (1, -1)]
    difference = (host(dy) * (y[0] - y[1])).sum() / (2 * t)
    size = np.abs(host(got["activations"]) * v).sum()
    # each element is rounded to its type (half a step), the difference itself is good to about t^2 and 1e-16 / t of its terms
    assert abs((host(got["activations"]) * v).sum() - difference) <= (ref.half_step(dtype) + 1e-4) * size + 1e-6


@pytest.mark.parametrize("c", [64, 128, 200, 384, 1025])
def test_encoded_output(dev, c):
    """The 8-bit output is the encoder's of the float32 output, bit for bit."""
    import localfold_b200 as lf
    x, g, b, _ = tensors(c, 70, c, "f32")
    plain = run(dev, x, g, b)["output"]
    both = run(dev, x, g, b, {"encode": "e4m3", "checkpoint": "e5m2"})
    want, kept = lf.float8_encode(dev, plain, 70, c), lf.float8_encode(dev, x, 70, c, {"format": "e5m2"})
    values = [lf.float8_decode(dev, t, {"output": "f32"}) for t in (both["output"], want, both["checkpoint"], kept)]
    dev.synchronize()
    assert torch.equal(values[0], values[1]) and torch.equal(values[2], values[3])


def test_special_rows(dev):
    """Constant rows, rows with infinities and not-a-numbers: each row only concerns itself, and the gradients' sums."""
    import localfold_b200 as lf
    x, g, b, rng = tensors(5, 40, 130, "f32")
    x[3] = 0
    x[4] = -2.5
    x[7, 5] = float("nan")
    x[9, 129] = float("inf")
    got = run(dev, x, g, b, {"statistics": True})
    dev.synchronize()
    with np.errstate(invalid="ignore"):
        want, mean, inverse = ref.layer_norm(host(x), host(g), host(b))
    good = np.isfinite(want).all(1)
    assert good.sum() == 38 and not np.isfinite(host(got["output"])[~good]).any()
    ref.close(got["output"][torch.as_tensor(good).cuda()], want[good], forward_bounds(host(x)[good], want[good], inverse[good], host(g), "f32"), "output")
    assert torch.equal(got["output"][3], b)
    dy = torch.zeros_like(x)
    dy[3:5] = 1
    back = lf.LayerNormGpu(dev).backward({"rows": 40, "channels": 130, "gradient": dy, "activations": x, "mean": got["mean"],
                                          "inverseDeviation": got["inverseDeviation"], "scale": g})
    dev.synchronize()
    dx = host(back["activations"])
    assert np.isnan(dx[7]).all() and np.isnan(dx[9]).all() and np.isfinite(dx[[i for i in range(40) if i not in (7, 9)]]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("c,shift", [(128, 1), (256, 3), (1536, 1), (96, 5)])
def test_any_address_and_in_place(dev, c, shift, dtype):
    """Tensors that start at any element give the bits of aligned ones; the output may be the input, the gradient's the gradient."""
    import localfold_b200 as lf
    rows = 70
    x, g, b, rng = tensors(c, rows, c, dtype)
    dy = torch.as_tensor(rng.standard_normal((rows, c))).to(TYPES[dtype]).cuda()

    def moved(t):
        room = torch.empty(t.numel() + 16, dtype=t.dtype, device="cuda")
        view = room[shift:shift + t.numel()].view(t.shape)
        view.copy_(t)
        return view

    layer = lf.LayerNormGpu(dev)
    want = run(dev, x, g, b, {"checkpoint": "e4m3"})
    xm, dym = moved(x), moved(dy)
    got = layer.run({"rows": rows, "channels": c, "activations": xm, "scale": moved(g), "offset": moved(b)}, {"checkpoint": "e4m3"}, out=xm)
    assert got["output"].data_ptr() == xm.data_ptr()
    rest = {"rows": rows, "channels": c, "scale": g}
    first = layer.backward({**rest, "gradient": dy, "activations": want["checkpoint"], "mean": want["mean"], "inverseDeviation": want["inverseDeviation"]})
    second = layer.backward({**rest, "gradient": dym, "activations": got["checkpoint"], "mean": got["mean"], "inverseDeviation": got["inverseDeviation"]}, out=dym)
    third = layer.backward({**rest, "gradient": dy, "activations": moved(x), "mean": want["mean"], "inverseDeviation": want["inverseDeviation"]})
    fourth = layer.backward({**rest, "gradient": dy, "activations": x, "mean": want["mean"], "inverseDeviation": want["inverseDeviation"]})
    dev.synchronize()
    assert torch.equal(xm, want["output"]) and torch.equal(dym, first["activations"])
    for a, b2 in ((first, second), (third, fourth)):
        for name in ("activations", "scale", "offset"):
            assert torch.equal(a[name], b2[name]), name
