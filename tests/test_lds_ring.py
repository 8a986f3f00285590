"""The barrier of a ring of LDS buffers, in the assembly that the build's flags give."""
import re
import shutil
import subprocess

import pytest

from relay_amd import build

SOURCE = """
#include "lds_ring.h"
// Reads a buffer, gives it back, and uses what it has read only afterwards.
extern "C" __global__ void give_back(const float* in, float* out) {
  __shared__ float buffer[2][64];
  buffer[0][threadIdx.x] = in[threadIdx.x];
  __syncthreads();
  const float read = buffer[0][threadIdx.x ^ 1];
  relay_hip::ring_barrier();
  buffer[0][threadIdx.x] = in[64 + threadIdx.x];
  out[threadIdx.x] = read;
}
"""


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="needs hipcc")
def test_reads_of_a_buffer_have_landed_before_the_barrier_that_frees_it(tmp_path):
    src, asm = tmp_path / "ring.hip", tmp_path / "ring.s"
    src.write_text(SOURCE)
    flags = [f for f in build.HIPCC_FLAGS if f != "-fPIC"]
    subprocess.run(["hipcc", *flags, "-I", build.CSRC, "--cuda-device-only", "-S", str(src), "-o", str(asm)], check=True, timeout=300, capture_output=True)
    body = asm.read_text().split("give_back:")[1].split("s_endpgm")[0]
    read = body.index("ds_read")
    between = body[read:body.index("s_barrier", read)]
    assert re.search(r"s_waitcnt [^\n]*lgkmcnt\(0\)", between), f"a read may still be under way at the barrier:\n{body}"
