"""The compiled walk over a paged cache: wait states of its MFMAs on accumulation registers and of its loads into LDS.  Runs without a GPU."""
import os
import shutil
import subprocess

from tests.test_key_side import OBJDUMP, _hazards
from vlm_training_amd import _lib


def test_inline_instructions_keep_their_wait_states(tmp_path):
    lib = shutil.copy(_lib.LIB_PATH, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, capture_output=True)
    count, kernels, found = 0, set(), []
    for name in sorted(os.listdir(tmp_path)):
        path = tmp_path / name
        held = {k for k in (b"dsa_paged_walk_kernelILi256", b"dsa_paged_walk_kernelILi128", b"dsa_paged_step_kernel") if name.endswith("gfx950") and k in path.read_bytes()}
        if held:
            kernels |= held
            c, f = _hazards(subprocess.run([OBJDUMP, "-d", str(path)], check=True, capture_output=True, text=True).stdout)
            count, found = count + c, found + f
    assert len(kernels) == 3 and count > 100 and not found, (kernels, count, found[:5])
