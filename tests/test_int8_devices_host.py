"""The products of up to 16 rows on several devices of one process, against a runtime that stands in for CUDA's: two devices, each
with limits of its own on a kernel's shared memory.  The library's object file is linked with it; no GPU."""
import os
import subprocess

import pytest

import tinyllama_c_b200  # noqa: F401  (the package's modules under its importable name)
from tinyllama_c_b200.csrc import build

CALLS = r"""
#include "gemm_int8.cuh"
#include <stdarg.h>

int tlc_int8_thin(const Int8Args& p, int out_dtype, cudaStream_t stream);
int g_tlc_pdl = 0;
int tlc_fail(int code, const char* fmt, ...) { va_list a; va_start(a, fmt); vprintf(fmt, a); va_end(a); printf("\n"); return code; }
void use_device(int d);
int launched();

int main() {
  Int8Args p = {};
  p.M = 16; p.N = 64; p.lda = p.ldw = p.K = 4096; p.ldo = 64;
  int bad = 0;
  for (int d : {0, 1, 0, 1, 70, 71})
    for (int out : {TLC_F32, TLC_BF16})
      for (int mode : {(int)I8_PLAIN, (int)I8_GLU}) {
        use_device(d);
        p.mode = mode;
        p.w_rows = mode == I8_GLU ? 128 : 64;
        bad += tlc_int8_thin(p, out, nullptr) != 0;
      }
  printf("%d launched, %d refused\n", launched(), bad);
  return bad || launched() != 24;
}
"""
RUNTIME = r"""
#include <cuda_runtime_api.h>
#include <map>
#include <utility>

static int device = 0, launches = 0;
static cudaError_t last = cudaSuccess;
static std::map<std::pair<int, const void*>, int> limit;          // bytes of dynamic shared memory, by device and kernel
void use_device(int d) { device = d; }
int launched() { return launches; }
extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute, int v) { limit[{device, f}] = v; return cudaSuccess; }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) {
  const int most = limit.count({device, f}) ? limit[{device, f}] : (48 - 16) * 1024;      // (16 KB are the kernel's static ones)
  if ((int)c->dynamicSmemBytes > most) return last = cudaErrorInvalidValue;
  launches++;
  return cudaSuccess;
}
cudaError_t cudaGetLastError() { const cudaError_t e = last; last = cudaSuccess; return e; }
const char* cudaGetErrorString(cudaError_t) { return "refused"; }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { return cudaErrorInvalidValue; }
// what the compiler's host code calls to make its kernels known
void** __cudaRegisterFatBinary(void*) { static void* h; return &h; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
char __cudaInitModule(void**) { return 0; }
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, void*) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return cudaSuccess; }
}
"""


def test_sixteen_rows_on_a_second_device(tmp_path):
    lib = build.build(verbose=False)
    obj = os.path.join(os.path.dirname(lib), "gemm_int8_thin.o")
    if not os.path.exists(obj):
        pytest.skip("the object files of the build are not here")
    (tmp_path / "calls.cu").write_text(CALLS)
    (tmp_path / "runtime.cpp").write_text(RUNTIME)
    exe = str(tmp_path / "calls")
    subprocess.run([build._nvcc(), *build._FLAGS, "-cudart", "none", "-I", build._HERE, str(tmp_path / "calls.cu"), str(tmp_path / "runtime.cpp"), obj,
                    "-o", exe], check=True)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout
