"""The training and 8-bit operators from their definitions in 64 bits (numpy), for the tests."""
import numpy as np

TOP = {"e4m3": 448.0, "e5m2": 57344.0}
BITS = {"e4m3": (3, -6), "e5m2": (2, -14)}      # mantissa bits, least normal exponent
U32 = 2.0 ** -24                                # half a step of float32, relative


def half_step(dtype):
    """A rounding to the type is off by at most this, relative to the value."""
    return {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}[dtype]


def exponents(x, block_rows=1, name="e4m3"):
    """log2 of each block's power of two: [row blocks][channel blocks]."""
    x = np.asarray(x, np.float64)
    rows, c = x.shape
    out = np.empty((-(-rows // block_rows), -(-c // 128)), np.int64)
    for i in range(out.shape[0]):
        for j in range(out.shape[1]):
            part = np.abs(x[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128])
            part = part[np.isfinite(part)]
            most = part.max() if part.size else 0.0
            e = -126
            if most > 0:
                mantissa, power = np.frexp(most)      # most = mantissa 2^power, mantissa < 1; TOP = 0.875 2^(9 or 16)
                e = max(-126, int(power) - (9 if name == "e4m3" else 16) + int(mantissa > 0.875))
            out[i, j] = e
    return out


def decoded(x, name="e4m3", block_rows=1):
    """The values that the 8-bit form stands for."""
    x = np.asarray(x, np.float64)
    rows, c = x.shape
    e = exponents(x, block_rows, name).repeat(block_rows, 0)[:rows].repeat(128, 1)[:, :c]
    bits, least = BITS[name]
    with np.errstate(invalid="ignore"):
        scaled = np.ldexp(x, -e)
        finite = np.where(np.isfinite(scaled), scaled, 0.0)
        _, power = np.frexp(finite)
        step = np.ldexp(1.0, np.maximum(power - 1, least) - bits)
        value = np.ldexp(np.rint(finite / step) * step, e)
    if name == "e4m3":
        return np.where(np.isfinite(x), value, np.nan)
    return np.where(np.isfinite(x), value, x)


def layer_norm(x, scale, offset, epsilon=1e-5):
    x = np.asarray(x, np.float64)
    mean = x.mean(1, keepdims=True)
    inverse = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + epsilon)
    return (x - mean) * inverse * scale + offset, mean[:, 0], inverse[:, 0]


def layer_norm_backward(dy, x, mean, inverse, scale):
    dy = np.asarray(dy, np.float64)
    u = (np.asarray(x, np.float64) - mean[:, None]) * inverse[:, None]
    h = dy * scale
    dx = inverse[:, None] * (h - h.mean(1, keepdims=True) - u * (h * u).mean(1, keepdims=True))
    return dx, (dy * u).sum(0), dy.sum(0)


def close(got, want, bound, what=""):
    """|got - want| <= bound everywhere, and not-a-number in the same places."""
    got = got.double().cpu().numpy() if hasattr(got, "cpu") else np.asarray(got, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: not-a-number in other places"
    with np.errstate(invalid="ignore"):
        far = np.where(got == want, 0.0, np.abs(got - want)) - bound
    far = np.nan_to_num(far, nan=-1.0, posinf=np.inf)
    assert (far <= 0).all(), f"{what}: beyond its bound by {far.max():.3e} at {np.unravel_index(far.argmax(), far.shape)}"
