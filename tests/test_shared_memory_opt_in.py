"""Dynamic shared memory beyond the default is asked for once a device for each kernel, also for kernels that share their parameters (host code against stand-ins for the two calls; no GPU needed)."""
import os
import subprocess

STAND_INS = r"""
#include <cuda_runtime_api.h>
int device, asked[2][2];
const void* second_kernel;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void* f, enum cudaFuncAttribute, int bytes) {
  ++asked[device][f == second_kernel];
  return bytes == (f == second_kernel ? 70000 : 60000) ? cudaSuccess : cudaErrorInvalidValue;
}
"""
MAIN = r"""
#include "linear_scan_host.cuh"
#include <stdio.h>
namespace ave { thread_local int g_last_cuda_error = 0; }
extern int device, asked[2][2];
extern const void* second_kernel;
static __global__ void first(int) {}
static __global__ void second(int) {}
int main() {
  second_kernel = (const void*)second;
  for (int turn = 0; turn < 2; ++turn)
    for (device = 0; device < 2; ++device)
      if (ave::allow_smem<&first>(60000) != 0 || ave::allow_smem<&second>(70000) != 0) return 1;
  device = 64;  // more than the library keeps notes of
  if (ave::allow_smem<&first>(60000) != AVE_GDN_UNSUPPORTED) return 2;
  printf("%d %d %d %d\n", asked[0][0], asked[0][1], asked[1][0], asked[1][1]);
}
"""


def test_every_kernel_is_asked_for_on_every_device(tmp_path):
    from avelang_b200 import build
    for name, text in (("main.cu", MAIN), ("stand_ins.cpp", STAND_INS)):
        (tmp_path / name).write_text(text)
    subprocess.run([build._nvcc(), *build.NVCC_FLAGS, "-cudart", "shared", "main.cu", "stand_ins.cpp", "-o", "main"], check=True, cwd=tmp_path)
    done = subprocess.run([os.path.join(tmp_path, "main")], capture_output=True, text=True, timeout=60)
    assert (done.returncode, done.stdout.split()) == (0, ["1"] * 4), done
