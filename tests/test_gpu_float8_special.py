"""Operands that hold infinities and values that are no numbers, and exponent bytes that belong to no row or block: neither reaches a result that it is not part of.

Bounds of finite results are those of ordinary operands: a float32 sum of K terms is off by at most K 2^-23 sum|terms| (additions may truncate)."""
import numpy as np
import pytest
import torch

import training_reference as ref

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -23
# few rows; tiles of 64, 128, 256 columns, many channels, pairs of multiprocessors; partial tiles, blocks and groups of 512 channels
SHAPES = [(3, 130, 72), (16, 384, 160), (200, 513, 100), (5000, 256, 1000), (300, 1030, 333), (129, 1200, 1001), (1999, 1155, 1537), (12001, 2048, 400), (700, 2048, 3000)]


@pytest.fixture(scope="module")
def dev():
    import localfold_b200 as lf
    d = lf.Device(0)
    yield d
    d.close()


def host(t):
    return t.double().cpu().numpy()


def poison(matrix):
    """Every exponent byte that belongs to no row or block becomes that of no number."""
    e, keep = matrix.exponents, torch.zeros_like(matrix.exponents, dtype=torch.bool)
    r, j = torch.meshgrid(torch.arange(matrix.rows, device="cuda"), torch.arange(-(-matrix.channels // 128), device="cuda"), indexing="ij")
    keep[j // 4, r // 128, r % 32, r % 128 // 32, j % 4] = True
    e[~keep] = 255
    return int((~keep).sum())


def spoil(t, rng, count):
    """``count`` values each that are no numbers, infinite, negatively infinite; two in the last row and column."""
    rows, c = t.shape
    for i, value in enumerate((float("nan"), float("inf"), float("-inf"))):
        r, k = rng.integers(0, rows, count), rng.integers(0, c, count)
        if i < 2:
            r[0], k[0] = rows - 1, c - 1 - i * (c > 1)
        t[torch.as_tensor(r).cuda(), torch.as_tensor(k).cuda()] = value
    return t


def compare(got, a, b, count, what):
    """``a @ b`` in 64 bits: the same places are infinite, no numbers, and finite within the bound of ``count`` terms."""
    with np.errstate(invalid="ignore", over="ignore"):
        want = a @ b
    got, finite = host(got), np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)]), what
    got, want = got[finite], want[finite]
    size = np.abs(np.where(np.isfinite(a), a, 0)) @ np.abs(np.where(np.isfinite(b), b, 0))
    assert (np.abs(got - want) <= count * STEP * size[finite]).all(), what


@pytest.mark.parametrize("name", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rows,c,n", SHAPES[:7])
def test_products(dev, rows, c, n, name):
    import localfold_b200 as lf
    rng = np.random.default_rng(rows + c)
    x = spoil(torch.as_tensor(rng.standard_normal((rows, c))).float().cuda(), rng, max(1, rows // 50))
    w, dy = (torch.as_tensor(rng.standard_normal(s)).float().cuda() for s in ((n, c), (rows, n)))
    spoil(dy, rng, max(1, rows // 50))
    linear, weights = lf.Float8LinearGpu(dev), lf.prepare_float8_linear_weights(dev, w)
    shape = {"rows": rows, "channels": c, "outChannels": n, "weights": weights}
    y = linear.run({**shape, "activations": x}, {"format": name, "checkpoint": True})
    dx = linear.input_gradient({**shape, "gradient": dy}, {"format": name})
    x8, dy8, w8 = ref.decoded(host(x), name), ref.decoded(host(dy), name), ref.decoded(host(w), "e4m3", 128)
    dev.synchronize()
    compare(y["output"], x8, w8.T, c, "output")
    compare(dx["output"], dy8, w8, n, "gradient")
    bad = w.clone()      # a weight with one of each
    bad[n // 2, c // 3], bad[n - 1, 0], bad[0, c - 1] = float("nan"), float("inf"), float("-inf")
    weights.update(bad)
    finite = torch.nan_to_num(x, nan=0.5, posinf=1.0, neginf=-1.0)
    y = linear.run({**shape, "activations": finite}, {"format": name})
    dev.synchronize()
    compare(y["output"], ref.decoded(host(finite), name), ref.decoded(host(bad), "e4m3", 128).T, c, "output of a weight that holds some")


@pytest.mark.parametrize("kind", ["bf16", "odd", "e4m3", "e5m2"])
@pytest.mark.parametrize("rows,c,n", [(1, 16, 8), (64, 128, 128), (100, 130, 72), (2100, 300, 256), (9000, 128, 2000)])
def test_weight_gradient(dev, rows, c, n, kind):
    import localfold_b200 as lf
    n += kind == "odd"
    rng = np.random.default_rng(rows + n)
    x = torch.as_tensor(rng.standard_normal((rows, c))).float().cuda()
    dy = torch.as_tensor(rng.standard_normal((rows, n))).bfloat16().cuda()
    chain = min(rows, 4096) / 16 + 16 + max(rows / 4096, 148)
    linear = lf.Float8LinearGpu(dev)
    for spoiled in ("gradient", "activations"):
        a, b = x.clone(), dy.clone()
        spoil(b if spoiled == "gradient" else a, rng, 1)
        x8 = lf.float8_encode(dev, a, rows, c, {"format": "e5m2"})
        operand = lf.float8_encode(dev, b, rows, n, {"format": kind}) if kind.startswith("e") else b
        got = linear.weight_gradient({"rows": rows, "channels": c, "outChannels": n, "gradient": operand, "activations": x8})
        dev.synchronize()
        av, bv = ref.decoded(host(a), "e5m2"), ref.decoded(host(b), kind) if kind.startswith("e") else host(b)
        compare(got["weight"], bv.T, av, chain, spoiled)
        compare(got["bias"][:, None], bv.T, np.ones((rows, 1)), chain, spoiled)


@pytest.mark.parametrize("rows,c,n", SHAPES)
def test_bytes_of_no_account(dev, rows, c, n):
    """Results are the same bits whatever the exponent bytes behind the last row and block are."""
    import localfold_b200 as lf
    torch.manual_seed(rows)
    x, dy, w = (torch.randn(s, device="cuda").bfloat16() for s in ((rows, c), (rows, n), (n, c)))
    linear, norm, weights = lf.Float8LinearGpu(dev), lf.LayerNormGpu(dev), lf.prepare_float8_linear_weights(dev, w)
    x8, dy8 = lf.float8_encode(dev, x, rows, c), lf.float8_encode(dev, dy, rows, n, {"format": "e5m2"})
    scale, mean, inverse = torch.rand(c, device="cuda"), torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    shape = {"rows": rows, "channels": c, "outChannels": n}

    def results():
        back = norm.backward({"rows": rows, "channels": c, "gradient": x, "activations": x8, "mean": mean, "inverseDeviation": inverse, "scale": scale})
        out = [linear.run({**shape, "activations": x8, "weights": weights})["output"], linear.input_gradient({**shape, "gradient": dy8, "weights": weights})["output"],
               lf.float8_decode(dev, x8), back["activations"], back["scale"], back["offset"]]
        for gradient in (dy, dy8):
            grads = linear.weight_gradient({**shape, "gradient": gradient, "activations": x8})
            out += [grads["weight"], grads["bias"]]
        dev.synchronize()
        return out

    before = results()
    assert poison(x8) > 0 and poison(dy8) > 0 and poison(weights.forward) + poison(weights.transposed) > 0
    for one, two in zip(before, results()):
        assert torch.isfinite(one).all() and torch.equal(one, two)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c", [(1, 8), (70, 64), (70, 128), (33, 200), (9, 1025), (300, 384)])
def test_encoded_output_e5m2(dev, rows, c, dtype):
    """LayerNorm's 8-bit output in e5m2: the code of the value before it is rounded to the activations' type."""
    import localfold_b200 as lf
    torch.manual_seed(c)
    x, g, b = torch.randn(rows, c, device="cuda").to(dtype), torch.rand(c, device="cuda") + 0.5, torch.randn(c, device="cuda")
    norm, call = lf.LayerNormGpu(dev), {"rows": rows, "channels": c, "scale": g, "offset": b}
    plain = norm.run({**call, "activations": x.float()})["output"]
    got = norm.run({**call, "activations": x}, {"encode": "e5m2", "checkpoint": "e4m3"})
    values = [lf.float8_decode(dev, t, {"output": "f32"}) for t in (got["output"], lf.float8_encode(dev, plain, rows, c, {"format": "e5m2"}), got["checkpoint"], lf.float8_encode(dev, x, rows, c))]
    dev.synchronize()
    assert got["output"].format == "e5m2" and got["checkpoint"].format == "e4m3"
    assert torch.equal(values[0], values[1]) and torch.equal(values[2], values[3])
