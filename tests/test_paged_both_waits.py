"""The compiled kernel of mixed batches over a paged cache (a file of its own, other flags, other template arguments than the kernels that it joins): the wait states of its inline
loads into LDS.  Runs without a GPU."""
import os
import shutil
import subprocess

from tests.test_key_side import OBJDUMP, _hazards
from vlm_training_amd import _lib

NAME = b"dsa_paged_both_kernel"


def test_loads_into_lds_keep_their_wait_states(tmp_path):
    lib = shutil.copy(_lib.LIB_PATH, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, capture_output=True)
    files = [p for p in sorted(os.listdir(tmp_path)) if p.endswith("gfx950") and NAME in (tmp_path / p).read_bytes()]
    assert len(files) == 1
    listing = subprocess.run([OBJDUMP, "-d", str(tmp_path / files[0])], check=True, capture_output=True, text=True).stdout
    # head_dim 64 and 128, bf16 and 8-bit; no MFMA on accumulation registers by name; every kernel asks for page numbers by loads into LDS, the bf16 ones for rows too
    functions = listing.split(">:\n")[1:]
    loads = [sum("offen lds" in line for line in f.splitlines()) for f in functions]
    assert len(functions) == 4 and min(loads) >= 2 and sum(n > 40 for n in loads) == 2, loads
    count, found = _hazards(listing)
    assert count == 0 and not found, (count, found[:5])
