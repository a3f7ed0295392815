"""Words around a 16-byte piece (csrc/hip/elements.h) come by loads whose whole address
the buffer's bounds check covers: the check of a raw buffer leaves the instruction's scalar
offset out, so that has to be 0 in every one of them."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

SOURCE = """
#include "elements.h"
using namespace spmm::engine::dev;
__global__ void pieces(const unsigned short* p, long long n, uint4* out) {
    const __amdgpu_buffer_rsrc_t buffer = words_buffer(p, n);
    const unsigned byte = threadIdx.x * 18u;
    out[threadIdx.x] = piece_of(load_words<true>(buffer, byte), byte);
    out[64 + threadIdx.x] = load_words<false>(buffer, byte).words;
}
"""


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason="no hipcc")
def test_loads_have_no_scalar_offset(tmp_path):
    src, asm = tmp_path / "pieces.hip", tmp_path / "pieces.s"
    src.write_text(SOURCE)
    subprocess.run([HIPCC, "-O3", "-std=c++17", "--offload-arch=gfx950", "--cuda-device-only", "-S",
                    "-I", os.path.join(ROOT, "sparse-matrix-multiplication_amd", "csrc", "hip"),
                    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", str(src), "-o",
                    str(asm)], check=True, capture_output=True)
    # buffer_load_dword v1, v2, s[0:3], <scalar offset> offen offset:16
    loads = re.findall(r"buffer_load_dword\S* \S+, \S+, s\[\d+:\d+\], (\S+) offen(?: offset:(\d+))?",
                       asm.read_text())
    # (the same four words by either load are read once)
    assert loads and sorted(o for _, o in loads)[-1] == "16", loads
    assert all(scalar == "0" for scalar, _ in loads), loads
