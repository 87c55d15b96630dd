"""A stand-in for the CUDA runtime on a machine without a GPU: the library's host side runs against it in a process of its own, and launches are only counted."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# (a null driver entry point would stop the tiled products at their tensor maps)
SOURCE = """
#include <stdlib.h>
#include <string.h>
static int launches, current;
static int map(void) { return 0; }
int fake_launches(void) { return launches; }
int cudaGetDeviceCount(int* n) { *n = 1; return 0; }
int cudaGetDevice(int* d) { *d = current; return 0; }
int cudaSetDevice(int d) { current = d; return 0; }
int cudaGetDeviceProperties_v2(void* p, int d) { return 1; }
int cudaGetDriverEntryPoint(const char* name, void** f, unsigned long long flags, int* found) { *f = (void*)map; *found = 0; return 0; }
int cudaFuncSetAttribute(const void* f, int a, int v) { return 0; }
int cudaGetLastError(void) { return 0; }
int cudaMalloc(void** p, size_t n) { *p = calloc(1, n); return 0; }
int cudaMallocHost(void** p, size_t n) { *p = calloc(1, n); return 0; }
int cudaFree(void* p) { free(p); return 0; }
int cudaFreeHost(void* p) { free(p); return 0; }
int cudaMemset(void* p, int v, size_t n) { memset(p, v, n); return 0; }
int cudaMemcpyAsync(void* to, const void* from, size_t n, int kind, void* s) { memcpy(to, from, n); return 0; }
int cudaStreamCreateWithFlags(void** s, unsigned f) { *s = calloc(1, 8); return 0; }
int cudaStreamDestroy(void* s) { free(s); return 0; }
int cudaStreamSynchronize(void* s) { return 0; }
int cudaStreamWaitEvent(void* s, void* e, unsigned f) { return 0; }
static void* capturing = (void*)-1;      /* the stream that is */
static int recorded;
void fake_capture(void* s) { capturing = s; }
int fake_recorded(void) { return recorded; }
int cudaStreamIsCapturing(void* s, int* status) { *status = s == capturing; return 0; }
int cudaEventCreate(void** e) { *e = calloc(1, 8); return 0; }
int cudaEventCreateWithFlags(void** e, unsigned f) { *e = calloc(1, 8); return 0; }
int cudaEventDestroy(void* e) { free(e); return 0; }
int cudaEventRecord(void* e, void* s) { ++recorded; return 0; }
int cudaLaunchKernelExC(const void* c, const void* f, void** a) { ++launches; return 0; }
"""
OPEN = """
import ctypes
from localfold_b200 import _native as nat
lib, context = nat.load(), ctypes.c_void_p()
assert lib.lf_context_create(0, None, ctypes.byref(context)) == nat.LF_OK
context, fake = context.value, ctypes.CDLL({fake!r})
launches = fake.fake_launches


def call(function, desc):
    # (status, message, launches)
    before = launches()
    status = getattr(lib, function)(context, ctypes.byref(desc), nat.Result())
    return status, lib.lf_last_error(context).decode() if status != nat.LF_OK else "", launches() - before

"""


def run(tmp_path, script):
    """``script`` after the lines above; what it prints."""
    source, fake = tmp_path / "fake.c", tmp_path / "fake.so"
    source.write_text(SOURCE)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(fake), str(source)], check=True)
    out = subprocess.run([sys.executable, "-c", OPEN.format(fake=str(fake)) + script], env={**os.environ, "LD_PRELOAD": str(fake), "PYTHONPATH": ROOT},
                         capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[-4000:]
    return out.stdout
