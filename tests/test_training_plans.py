"""The sizes of the training operators' workspaces and plans at the ends of their ranges: host arithmetic, without a GPU.

The functions read one number of a context, its multiprocessors: a buffer that says 148 everywhere stands for it.  Each runs in a process of its own,
since a division by zero ends one."""
import os
import subprocess
import sys

import pytest

import localfold_b200 as lf
from test_training_refusals import DEVICE, Fake, float8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ASK = """
import ctypes, sys
from localfold_b200 import _native as nat
lib = nat.load()
context = (ctypes.c_int32 * 16384)(*[148] * 16384)
name, *sizes = sys.argv[1:]
arguments = [int(s) for s in sizes]
if name != "lf_float8_linear_workspace":
    arguments.insert(0, ctypes.addressof(context))
print(getattr(lib, name)(*arguments))
"""


def ask(name, *sizes):
    out = subprocess.run([sys.executable, "-c", ASK, name, *map(str, sizes)], capture_output=True, text=True, env={**os.environ, "PYTHONPATH": ROOT})
    assert out.returncode == 0, (name, sizes, out.returncode, out.stderr)
    return int(out.stdout)


@pytest.mark.parametrize("rows,channels,outputs", [(1, 1 << 22, 1 << 26), (1, 1 << 22, 1 << 25), (1, (1 << 22) + 1, 8), (1, 8, (1 << 22) + 1), (1, 2 ** 31 - 1, 2 ** 31 - 1), (64, 1 << 24, 1 << 24), (2 ** 31 - 1, 8, 8)])
def test_no_workspace_beyond_the_limits(rows, channels, outputs):
    assert ask("lf_float8_weight_gradient_workspace", rows, channels, outputs) == 0


def test_workspace_at_the_limits():
    assert ask("lf_float8_weight_gradient_workspace", 64, 1 << 22, 1 << 22) == 0      # one split: the products are the gradient
    assert ask("lf_float8_weight_gradient_workspace", 148 * 256, 128, 128) == 148 * 128 * 129 * 4


@pytest.mark.parametrize("rows", [64 * 65535 * 64 + 1, 1_860_000_000, 1_859_838_912 + 64 * 148, 2_000_000_000, 2 ** 31 - 257, 2 ** 31 - 256])
@pytest.mark.parametrize("channels,outputs", [(8, 8), (8, 128), (256, 300)])
def test_splits_fit_the_grid(rows, channels, outputs):
    size = outputs * (channels + 1) * 4
    nbytes = ask("lf_float8_weight_gradient_workspace", rows, channels, outputs)
    assert nbytes % size == 0 and 148 < nbytes // size <= 65535


def test_splits_over_the_whole_range():
    """... and at every 64th thousand of rows, in one process."""
    many = ASK.replace("print(getattr(lib, name)(*arguments))", "call = getattr(lib, name)\n"
                       "print(max(call(arguments[0], rows, 8, 8) for rows in range(1 << 20, 2 ** 31 - 256, 64000)) // (8 * 9 * 4))")
    out = subprocess.run([sys.executable, "-c", many, "lf_float8_weight_gradient_workspace"], capture_output=True, text=True, env={**os.environ, "PYTHONPATH": ROOT})
    assert out.returncode == 0 and 60000 < int(out.stdout) <= 65535, (out.stdout, out.stderr)


@pytest.mark.parametrize("rows,channels", [(17, 2 ** 31 - 1), (17, 2 ** 31 - 16), (100, 1 << 24), (2 ** 31 - 1, 8)])
def test_bytes_of_an_operand(rows, channels):
    codes = rows * (-(-channels // 16) * 16)
    assert ask("lf_float8_linear_workspace", rows, channels) == codes + -(-channels // 512) * -(-rows // 128) * 512


@pytest.mark.parametrize("channels,outputs", [(1 << 22, 1 << 25), ((1 << 22) + 1, 8), (8, (1 << 22) + 1)])
def test_refused_before_memory_is_asked_for(channels, outputs):
    call = {"rows": 1, "channels": channels, "outChannels": outputs, "activations": float8(1, channels), "gradient": Fake(outputs)}
    with pytest.raises(NotImplementedError, match=f"the weight's gradient of {outputs} x {channels} channels: at most 4194304 of either"):
        lf.Float8LinearGpu(DEVICE).weight_gradient(call)
