"""Results that overlap operands: refused at every size alike, but where a call says that it works in place."""
import pytest
import torch

import fake_cuda

# Addresses are only compared: nothing is launched.  x, w: codes and exponents of 4 x 8 and 8 x 8 (or of many rows), 4096 bytes apart at least.
SCRIPT = """
A = nat.LF_ERR_ARGUMENT


def matrix(rows, channels, codes, exponents=None):
    return nat.Float8Matrix(rows, channels, 0, codes, exponents or codes and codes + (rows * 16 + 4095) // 4096 * 4096)


def refused(function, desc):
    status, text, launched = call(function, desc)
    assert status == A and "the output overlaps an operand" in text and launched == 0, (function, status, text)


def taken(function, desc):
    status, text, launched = call(function, desc)
    assert status == nat.LF_OK and launched > 0, (function, status, text)


BASE = 1 << 32
for rows in (1, 4, 16, 17, 5000):
    for dtype, size in ((0, 4), (1, 2)):
        x, w, ones, out, room = (BASE + (i << 24) for i in range(5))
        n = c = 8
        whole = rows * c * size
        lin = lambda out, **k: nat.Float8LinearDesc(**{**dict(activations=matrix(rows, c, None), weights=matrix(n, c, w), bias=ones, out_dtype=dtype, source_dtype=dtype, source=x, out=out,
                                                               workspace=room, workspace_bytes=1 << 24), **k})
        taken("lf_float8_linear_run", lin(out))
        taken("lf_float8_linear_run", lin(x + whole))
        taken("lf_float8_linear_run", lin(x - whole))
        for at in (x, x + size, x + whole - size, x - whole + size, w, w + 64, matrix(n, c, w).exponents, ones, ones + 4 * n - size):
            refused("lf_float8_linear_run", lin(at))
        if rows > 16:
            refused("lf_float8_linear_run", lin(room + 32))
        kept = matrix(rows, c, room)
        taken("lf_float8_linear_run", lin(out, activations=kept))
        taken("lf_float8_linear_run", lin(out, activations=kept, source=None))
        for source in (None, x):
            for at in (kept.codes, kept.exponents, kept.exponents + 256):
                refused("lf_float8_linear_run", lin(at, activations=kept, source=source))

        decode = lambda out: nat.Float8DecodeDesc(kept, dtype, 0, out)
        taken("lf_float8_decode", decode(out))
        for at in (kept.codes, kept.codes + 16 * rows - 8, kept.exponents):
            refused("lf_float8_decode", decode(at))

        norm = lambda out: nat.LayerNormDesc(rows=rows, channels=c, variance=1, act_dtype=dtype, epsilon=1e-5, activations=x, scale=ones, offset=ones + (1 << 20), out=out)
        back = lambda out, **k: nat.LayerNormBackwardDesc(**{**dict(rows=rows, channels=c, act_dtype=dtype, gradient=x, activations=w, mean=ones, inverse_deviation=ones + (1 << 20), scale=ones + (1 << 21), out=out,
                                                                     scale_gradient=ones + (1 << 22), offset_gradient=ones + (1 << 23), workspace=room, workspace_bytes=1 << 24), **k})
        taken("lf_layer_norm_run", norm(out))
        taken("lf_layer_norm_run", norm(x))
        for at in (x + size, x - size, x + whole - size, ones, ones + 4 * c - size, ones + (1 << 20) + 4):
            refused("lf_layer_norm_run", norm(at))
        for at in (out, x, w):
            taken("lf_layer_norm_backward_run", back(at))
        for at in (x + size, x - size, w + size, w + whole - size, ones, ones + 4 * rows - size, ones + (1 << 20), ones + (1 << 21) + 4):
            refused("lf_layer_norm_backward_run", back(at))
        kept = matrix(rows, c, w)
        taken("lf_layer_norm_backward_run", back(x, activations=None, checkpoint=kept))
        for at in (kept.codes, kept.exponents):
            refused("lf_layer_norm_backward_run", back(at, activations=None, checkpoint=kept))
print("done")
"""


def test_library(tmp_path):
    assert fake_cuda.run(tmp_path, SCRIPT).split() == ["done"]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 16, 17, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_package(rows, dtype):
    import localfold_b200 as lf
    c = 64
    d = lf.Device(0)
    room = torch.randn(3 * rows * c, device="cuda").to(dtype)
    x, scale = room[:rows * c].view(rows, c), torch.rand(c, device="cuda")
    shifted = room[8:8 + rows * c].view(rows, c)
    before = room.clone()
    linear, norm, weights = lf.Float8LinearGpu(d), lf.LayerNormGpu(d), lf.prepare_float8_linear_weights(d, torch.randn(c, c, device="cuda"))
    call, shape = {"rows": rows, "channels": c, "outChannels": c, "weights": weights}, {"rows": rows, "channels": c, "scale": scale}
    stats = norm.run({**shape, "activations": x, "offset": scale}, {"statistics": True})
    back = {**shape, "mean": stats["mean"], "inverseDeviation": stats["inverseDeviation"]}
    apart = torch.empty_like(x)
    want = norm.backward({**back, "gradient": x, "activations": shifted})["activations"]
    for out in (x, shifted):
        for refused in (lambda: linear.run({**call, "activations": x}, None, out), lambda: linear.input_gradient({**call, "gradient": x}, None, out)):
            with pytest.raises(ValueError, match="the output overlaps an operand"):
                refused()
    for refused in (lambda: norm.run({**shape, "activations": x, "offset": scale}, None, shifted), lambda: norm.backward({**back, "gradient": x, "activations": x}, None, shifted)):
        with pytest.raises(ValueError, match="the output overlaps an operand"):
            refused()
    d.synchronize()
    assert torch.equal(room, before)
    # the activations may be the result's place, too
    got = norm.backward({**back, "gradient": x, "activations": apart.copy_(shifted)}, None, apart)["activations"]
    d.synchronize()
    assert got.data_ptr() == apart.data_ptr() and torch.equal(apart, want)
    d.close()
