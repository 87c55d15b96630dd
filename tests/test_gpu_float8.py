"""The 8-bit form of a matrix: encoder and decoder, bit for bit against the definition."""
import numpy as np
import pytest
import torch

import training_reference as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SHAPES = [(1, 1), (2, 7), (1, 16), (129, 8), (63, 64), (70, 65), (257, 128), (5, 129), (31, 200), (40, 384), (9, 513), (3, 1155), (130, 4096), (5000, 24)]


@pytest.fixture(scope="module")
def dev():
    import localfold_b200 as lf
    d = lf.Device(0)
    yield d
    d.close()


def matrix(seed, rows, c, dtype):
    """Every binary order of magnitude, values next to the codes' borders, zeros."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, c)) * np.exp2(rng.integers(-30, 30, (rows, c)) * (rng.random((rows, 1)) < 0.3)) * np.exp2(rng.integers(-90, 90, (rows, 1)))
    ties = np.rint(x / np.exp2(np.floor(np.log2(np.abs(x))) - 4)) * np.exp2(np.floor(np.log2(np.abs(x))) - 4)      # halfway between codes, or codes
    x = np.where(rng.random((rows, c)) < 0.3, ties, x)
    x[rng.random((rows, c)) < 0.1] = 0
    x[rng.random(rows) < 0.05] = 0
    return torch.as_tensor(x).to(TYPES[dtype]).cuda()


def host(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("name", ["e4m3", "e5m2"])
@pytest.mark.parametrize("rows,c", SHAPES)
def test_round_trip(dev, rows, c, name, dtype):
    import localfold_b200 as lf
    x = matrix(rows * 100 + c, rows, c, dtype)
    kept = lf.float8_encode(dev, x, rows, c, {"format": name})
    got = {out: lf.float8_decode(dev, kept, {"output": out}) for out in TYPES}
    dev.synchronize()
    want = ref.decoded(host(x), name)
    for out in TYPES:
        assert got[out].dtype == TYPES[out]
        ref.close(got[out], want, 0.0, out)
    e = kept.exponents.cpu().numpy().astype(np.int64)
    r, j = np.meshgrid(np.arange(rows), np.arange(-(-c // 128)), indexing="ij")
    assert np.array_equal(e[j // 4, r // 128, r % 32, r % 128 // 32, j % 4] - 127, ref.exponents(host(x), 1, name))
    assert not kept.codes[:, c:].any()
    assert kept.nbytes <= rows * (c + 15) + 512 * -(-rows // 128) * -(-c // 512)


@pytest.mark.parametrize("name", ["e4m3", "e5m2"])
def test_special_values(dev, name):
    """Values that are not finite have no say in the scale; the largest and smallest floats and negative zeros survive."""
    import localfold_b200 as lf
    x = torch.randn(12, 200, device="cuda")
    x[0, 5], x[1, 6], x[2, 130] = float("nan"), float("inf"), float("-inf")
    x[3] = float("nan")
    x[4] = float("inf")
    x[5] = 2.0 ** -149
    x[6], x[6, 0] = 1e-40, 2.0 ** -126
    x[7] = 3.0e38
    x[8] = -0.0
    x[9, :4] = torch.tensor([448.0, 449.0, 464.0, 480.0])
    x[10, :2] = torch.tensor([57344.0, 57345.0])
    x[11] *= 2.0 ** -120
    got = lf.float8_decode(dev, lf.float8_encode(dev, x, 12, 200, {"format": name}), {"output": "f32"})
    dev.synchronize()
    ref.close(got, ref.decoded(host(x), name), 0.0, name)
    assert torch.signbit(got[8]).all()


@pytest.mark.parametrize("name", ["e4m3", "e5m2"])
def test_least_values(dev, name):
    """Blocks whose codes lie beneath bf16's least step: exact in float32, rounded to nearest in bf16."""
    import localfold_b200 as lf
    x = torch.as_tensor(np.ldexp(np.random.default_rng(5).standard_normal((40, 300)), np.arange(-145, -105)[:, None])).float().cuda()
    kept = lf.float8_encode(dev, x, 40, 300, {"format": name})
    exact, rounded = (lf.float8_decode(dev, kept, {"output": out}) for out in ("f32", "bf16"))
    dev.synchronize()
    ref.close(exact, ref.decoded(host(x), name), 0.0, "f32")
    ref.close(rounded, host(exact.bfloat16()), 0.0, "bf16")
    assert (rounded.float() != exact).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [1, 2, 3, 8])
def test_any_address(dev, shift, dtype):
    import localfold_b200 as lf
    x = matrix(shift, 37, 256, dtype)
    room = torch.empty(x.numel() + 16, dtype=x.dtype, device="cuda")
    view = room[shift:shift + x.numel()].view(x.shape)
    view.copy_(x)
    a, b = lf.float8_encode(dev, x, 37, 256), lf.float8_encode(dev, view, 37, 256)
    out = torch.empty(x.numel() + 16, dtype=x.dtype, device="cuda")
    out.fill_(7)
    lf.float8_decode(dev, a, {"output": dtype}, out=out[shift:shift + x.numel()].view(x.shape))
    again = lf.float8_decode(dev, b, {"output": dtype})
    dev.synchronize()
    assert torch.equal(a.codes, b.codes) and torch.equal(out[shift:shift + x.numel()].view(x.shape), again)
    assert (out[:shift] == 7).all() and (out[shift + x.numel():] == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,c", [(1, 1), (5, 3), (128, 128), (130, 64), (64, 300), (384, 129), (257, 1000)])
def test_weights(dev, n, c, dtype):
    """One exponent for 128 x 128 elements, the same values in both orientations; update() replaces them."""
    import localfold_b200 as lf
    for seed in (1, 2):
        w = matrix(seed * 1000 + n + c, n, c, dtype)
        if seed == 2:
            w[n // 2, c // 2] = float("nan")
        if seed == 1:
            weights = lf.prepare_float8_linear_weights(dev, w)
        else:
            weights.update(w)
        got = lf.float8_decode(dev, weights.forward, {"output": "f32"})
        turned = lf.float8_decode(dev, weights.transposed, {"output": "f32"})
        dev.synchronize()
        want = ref.decoded(host(w), "e4m3", 128)
        ref.close(got, want, 0.0, "forward")
        ref.close(turned, want.T, 0.0, "transposed")
        assert not weights.forward.codes[:, c:].any() and not weights.transposed.codes[:, n:].any()
