"""The wait of the kernels' inner loops ends by itself: at the time limit, and at once when another wait of its block has run out."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from triton_b200.build import CSRC, NVCC_FLAGS

PROBE = r"""
#include "gemm_tc_common.cuh"
// a barrier at which nobody arrives; took: the wait's cycles, status: what it reports
__global__ void probe_kernel(int aborted, long long* took, int32_t* status) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ int abort;
  if (threadIdx.x == 0) { mbar_init(smem_u32(&bar), 1); abort = aborted; }
  __syncthreads();
  const Ctl ctl{&abort, status};
  const long long t0 = clock64();
  mbar_wait_short(smem_u32(&bar), 0, ctl, 1002);
  if (threadIdx.x == 0) { took[0] = clock64() - t0; took[1] = WAIT_LIMIT_CYCLES; took[2] = abort; }
}
extern "C" int probe(int aborted, long long* took, int32_t* status, void* stream) {
  probe_kernel<<<1, 32, 0, (cudaStream_t)stream>>>(aborted, took, status);
  return (int)cudaGetLastError();
}
"""


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        pytest.skip("no nvcc")
    where = tmp_path_factory.mktemp("probe")
    (where / "probe.cu").write_text(PROBE)
    flags = [f for f in NVCC_FLAGS if f not in ("-Xcompiler", "-fvisibility=hidden", "-fPIC")]
    subprocess.run([nvcc, *flags, "-Xcompiler", "-fPIC", "-shared", "-I", str(CSRC), str(where / "probe.cu"), "-o", str(where / "probe.so")], check=True)
    lib = ctypes.CDLL(str(where / "probe.so"))
    lib.probe.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
    return lib.probe


def test_the_wait_compiles_by_itself(probe):
    assert probe is not None


@pytest.mark.gpu
@pytest.mark.parametrize("aborted", [0, 1])
def test_a_wait_for_nothing_ends(probe, aborted):
    took, status = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert probe(aborted, took.data_ptr(), status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    cycles, limit, abort = took.tolist()
    assert abort == 1
    if aborted:
        assert status.item() == 0 and cycles < limit // 8
    else:
        assert status.item() == 1002 and limit < cycles < limit + limit // 8
