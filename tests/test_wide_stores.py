"""A buffer store of 16 bytes must not be followed at once by an instruction that overwrites what it stores.  With a scalar register as its offset the
compiler leaves that wait state out, and the stored values were wrong now and then: no such store in the assembly of the delta-rule kernels."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vlm_training_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
@pytest.mark.parametrize("name", ["dsa_delta_walk", "dsa_delta_chain"])
def test_wide_buffer_stores_have_no_scalar_offset(name, tmp_path):
    out = tmp_path / "k.s"
    subprocess.run([HIPCC, "-O3", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-w", "--cuda-device-only", "-S",
                    os.path.join(CSRC, name + ".hip"), "-o", str(out)], check=True, capture_output=True)
    stores = re.findall(r"^\s*buffer_store_dwordx[34] .*$", out.read_text(), re.M)
    assert stores
    for line in stores:
        offset = line.split("],")[-1].split()[0]
        assert offset == "0", line
