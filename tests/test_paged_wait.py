"""The bounded wait of the paged attention answers for a whole warp: when the limit runs out for some of
its lanes, all of them are told so, and the error word says which wait it was.

A kernel of one warp is built from the header for it. Half of the lanes wait for a barrier whose phase is
complete, the other half for one that nothing ever completes, for the kernels' limit of 2 s; nothing
faults or spins without bound, and the context stays usable."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

SOURCE = r"""
#include "paged_attn.cuh"
__global__ void waits(int* answer, int* err) {
  __shared__ uint64_t bar[2];
  if (threadIdx.x == 0) {
    nk::mbar_init(&bar[0], 1);
    nk::mbar_init(&bar[1], 1);
    nk::fence_barrier_init();
    nk::mbar_arrive(&bar[0]);
  }
  __syncwarp();
  answer[threadIdx.x] = nk::pa::wait(&bar[0], 0, nk::kErrTimeoutOther, err);
  __syncwarp();
  answer[32 + threadIdx.x] = nk::pa::wait(&bar[threadIdx.x & 1], 0, nk::kErrTimeoutMma, err);
}
extern "C" int run_waits(int* answer, int* err) {
  waits<<<1, 32>>>(answer, err);
  const cudaError_t launched = cudaGetLastError();
  return launched != cudaSuccess ? int(launched) : int(cudaDeviceSynchronize());
}
"""


@pytest.mark.gpu
def test_a_wait_that_runs_out_for_some_lanes_runs_out_for_all(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    kernels = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc", "kernels")
    source, lib = tmp_path / "waits.cu", tmp_path / "waits.so"
    source.write_text(SOURCE)
    subprocess.run([nvcc, "-shared", "-Xcompiler", "-fPIC", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a",
                    "-I", kernels, "-o", str(lib), str(source)], check=True)
    run = ctypes.CDLL(str(lib)).run_waits
    run.argtypes = [ctypes.c_void_p] * 2
    answer = torch.full((64,), -1, device="cuda", dtype=torch.int32)
    err = torch.zeros(1, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    assert run(answer.data_ptr(), err.data_ptr()) == 0
    assert answer.tolist() == [1] * 32 + [0] * 32
    assert err.item() == 2  # the code of the second wait
    assert float((torch.ones(64, device="cuda") * 2).sum()) == 128.0
