"""A HIP runtime that runs nothing, for tests of what happens in front of a launch: it comes before the real one in a process of its own, so nothing here needs a GPU.

Two devices unless devices(n) says otherwise: device 1 holds the addresses from 2^40 on and the streams with odd handles, addresses below 2^16 are no device's.  Launches are counted; a grid that
the real runtime refuses (2^32 threads and more along x, no blocks) is an error and counted apart."""
import os
import subprocess
import sys

import ngp_abi as A

RUNTIME = r"""
#include <hip/hip_runtime_api.h>
#include <stdint.h>
#include <string.h>
static int n_devices = 2, launched, too_large;
extern "C" {
hipError_t hipGetDeviceCount(int* n) { *n = n_devices; return hipSuccess; }
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipStreamGetDevice(hipStream_t s, hipDevice_t* d) { *d = (int)((uintptr_t)s & 1); return hipSuccess; }
hipError_t hipPointerGetAttributes(hipPointerAttribute_t* a, const void* p) {
	memset(a, 0, sizeof(*a));
	if ((uintptr_t)p < 0x10000) return hipErrorInvalidValue;
	a->type = hipMemoryTypeDevice; a->device = (uintptr_t)p >> 40 ? 1 : 0;
	return hipSuccess;
}
static hipError_t last = hipSuccess;
hipError_t hipGetLastError(void) { hipError_t e = last; last = hipSuccess; return e; }
static dim3 grid_, block_;
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t, hipStream_t) { grid_ = grid; block_ = block; return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* s) { *grid = grid_; *block = block_; *lds = 0; *s = nullptr; return hipSuccess; }
hipError_t hipLaunchKernel(const void*, dim3 grid, dim3 block, void**, size_t, hipStream_t) {
	if (!grid.x || !grid.y || !grid.z || (uint64_t)grid.x * block.x >> 32 || grid.y > 65535 || grid.z > 65535) { ++too_large; return last = hipErrorInvalidConfiguration; }
	++launched; return hipSuccess;
}
void devices(int n) { n_devices = n; }
int launches(void) { return launched; }
int launches_out_of_range(void) { return too_large; }
}
"""

HEAD = """
import ctypes as C, sys
runtime = C.CDLL(sys.argv[1], C.RTLD_GLOBAL)
import ngp_abi as A
L = A.load_hip()
"""


def run(code, tmp_path):
    """`code` in a process whose library calls this runtime (`runtime`; the library is `L`); it ends by printing: done"""
    source, library = tmp_path / "runtime.cpp", tmp_path / "libruntime.so"
    source.write_text(RUNTIME)
    subprocess.check_call(["g++", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", str(source), "-o", str(library)])
    path = os.pathsep.join([os.path.dirname(os.path.abspath(A.__file__)), os.environ.get("PYTHONPATH", "")])
    r = subprocess.run([sys.executable, "-c", HEAD + code, str(library)], env={**os.environ, "PYTHONPATH": path}, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]
