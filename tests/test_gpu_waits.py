"""A bounded wait that runs out: the barrier helpers return, and the status says so.

A kernel of the test's own waits, with a short limit, on a barrier that nobody
arrives at; the flag goes the way of the operators' (gs_*_status)."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

CSRC = Path(__file__).resolve().parent.parent / "gaussian-splats_b200" / "csrc"
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

SOURCE = r"""
#include "tensorcore.cuh"
namespace gs { void set_cuda_error(cudaError_t) {} }
__device__ uint32_t g_flag;
__global__ void wait_kernel(int arrive, int* out) {
  __shared__ uint64_t bar;
  const uint32_t b = gs::tc::shared_address(&bar);
  if (threadIdx.x == 0) {
    gs::tc::barrier_init(b, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (arrive) gs::tc::barrier_arrive(b);
  }
  __syncthreads();
  const bool good = gs::tc::barrier_wait(b, 0, 100);
  if (!good && threadIdx.x == 0) {
    gs::tc::barrier_settle(b);
    atomicExch(&g_flag, 1u);
  }
  if (threadIdx.x == 0) *out = good;
}
extern "C" int wait_and_ask(int arrive, int* came) {
  int* out;
  if (cudaMalloc(&out, sizeof(int))) return -100;
  wait_kernel<<<1, 32>>>(arrive, out);
  const int status = gs::take_timeout(g_flag, nullptr);
  if (cudaMemcpy(came, out, sizeof(int), cudaMemcpyDeviceToHost)) return -100;
  cudaFree(out);
  return status;
}
"""


@pytest.mark.skipif(not Path(NVCC).exists(), reason="no nvcc")
def test_a_wait_that_runs_out_is_told(tmp_path):
    import torch

    (tmp_path / "wait.cu").write_text(SOURCE)
    library = tmp_path / "wait.so"
    subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-shared",
                    "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", f"-I{CSRC}",
                    str(tmp_path / "wait.cu"), "-o", str(library)], check=True)
    torch.cuda.synchronize()
    lib, came = ctypes.CDLL(str(library)), ctypes.c_int()
    timeout = -6  # GS_ERR_TIMEOUT
    for arrive, status in ((1, 0), (0, timeout), (1, 0), (0, timeout), (1, 0)):
        assert lib.wait_and_ask(arrive, ctypes.byref(came)) == status
        assert came.value == arrive
