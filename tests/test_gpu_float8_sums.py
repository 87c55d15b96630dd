"""The bias' gradient beside the weight's, in blocks of few steps: the sums of dy are taken from shared memory that the output's tiles go through afterwards.

Gradients and activations are small whole numbers: exact in bf16 and in e4m3 (at most 8, four significant bits), and so are all sums (below 2^24)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    import localfold_b200 as lf
    d = lf.Device(0)
    yield d
    d.close()


# one step of 64 rows to seven, few channels (short products), one block of 128 outputs a tile and, from 2^31 multiplications on, two
@pytest.mark.parametrize("mode", ["whole", "odd", "codes"])
@pytest.mark.parametrize("rows,c,n", [(1, 8, 128), (64, 8, 128), (64, 64, 1024), (100, 16, 256), (192, 64, 4096), (448, 33, 136), (64, 64, 1 << 19), (192, 64, 1 << 18),
                                      (128, 128, 140000), (320, 200, 80000)])
def test_bias(dev, rows, c, n, mode):
    import localfold_b200 as lf
    n += mode == "odd"      # (rows that no 16-byte access divides)
    torch.manual_seed(rows + c)
    x = torch.randint(-8, 9, (rows, c), device="cuda").float()
    dy = torch.randint(-8, 9, (rows, n), device="cuda").bfloat16()
    x[:, 0] = 8
    want, sums = (dy.double().T @ x.double()).float(), dy.double().sum(0).float()
    x8 = lf.float8_encode(dev, x, rows, c)
    gradient = lf.float8_encode(dev, dy, rows, n) if mode == "codes" else dy
    linear, call = lf.Float8LinearGpu(dev), {"rows": rows, "channels": c, "outChannels": n, "activations": x8, "gradient": gradient}
    for _ in range(10):
        got = linear.weight_gradient(call)
        dev.synchronize()
        assert torch.equal(got["bias"], sums) and torch.equal(got["weight"], want)
