"""Calls leave the thread's current GPU as it was."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# CUDA's answers for a machine of two GPUs, as far as the call asks
FAKE = """
static int current = 1;
int cudaGetDevice(int* d) { *d = current; return 0; }
int cudaSetDevice(int d) { current = d; return 0; }
int cudaEventRecord(void* e, void* s) { return current == 0 ? 0 : 400; }
int cudaStreamWaitEvent(void* s, void* e, unsigned f) { return current == 0 ? 0 : 400; }
int fake_current(void) { return current; }
"""
CALL = """
import ctypes
from localfold_b200 import _native as nat
fake, lib = ctypes.CDLL({fake!r}), nat.load()
context = ctypes.create_string_buffer(1 << 16)      # (GPU 0, CUDA's default stream)
assert fake.fake_current() == 1
assert lib.lf_context_await(ctypes.addressof(context), 64) == nat.LF_OK
print("current", fake.fake_current())
"""


def test_await_restores_the_current_gpu(tmp_path):
    """The event is recorded with the context's GPU current, and the caller's is current again afterwards."""
    source, fake = tmp_path / "fake.c", tmp_path / "fake.so"
    source.write_text(FAKE)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(fake), str(source)], check=True)
    env = {**os.environ, "LD_PRELOAD": str(fake), "PYTHONPATH": ROOT}
    out = subprocess.run([sys.executable, "-c", CALL.format(fake=str(fake))], env=env, capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    assert out.stdout.split() == ["current", "1"]


@pytest.mark.gpu
def test_operators_restore_the_current_gpu():
    import torch
    import localfold_b200 as lf
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    d = lf.Device(0)
    torch.cuda.set_device(1)
    try:
        x = torch.randn(8, 64, device="cuda:0")
        lf.float8_decode(d, lf.float8_encode(d, x, 8, 64))
        assert torch.cuda.current_device() == 1
    finally:
        torch.cuda.set_device(0)
        d.close()
