"""Paged attention over more blocks than a launch has room for is refused: 2^32 threads and more along x are cut to 32 bits without an error.  Runs without a GPU."""
import pytest

from tests.test_cache_refusals import _args
from vlm_training_amd import _lib


def _call(T, N, Hkv, new, longest):
    lib = _lib.load()
    cache = _args(Hkv=Hkv, k_page=Hkv * 64 * 128, v_page=Hkv * 64 * 128)
    code = lib.dsa_paged_attn(cache, 16, 512, 128, 16, 16, T, N, 2 * Hkv, 1.0, new, longest, 16, None, None, 0, None)
    return code, lib.dsa_last_error(), lib.dsa_paged_attn_workspace_bytes(cache, T, N, 2 * Hkv, new, longest)


# (a workgroup of 256 threads to each block and kv head: 2^24 - 1 of them fit)
@pytest.mark.parametrize("T,N,Hkv,new,longest", [(1 << 24, 1 << 24, 1, 1, 0), (1 << 23, 1 << 23, 2, 1, 400), ((1 << 24) + 5, 1 << 24, 1, 7, 0), ((1 << 27) - 1, 1 << 25, 8, 0, 0),
                                                 (1 << 30, 1, 1, 0, 0)])
def test_more_blocks_than_fit(T, N, Hkv, new, longest):
    code, error, need = _call(T, N, Hkv, new, longest)
    assert code == -2 and b"too many" in error and need == 0, (code, error, need)


# the same with room: what is missing is the workspace
@pytest.mark.parametrize("T,N,Hkv,new", [((1 << 24) - 1, (1 << 24) - 1, 1, 1), ((1 << 23) - 1, (1 << 23) - 1, 2, 1), (1 << 28, 2, 1, 0)])
def test_as_many_as_fit(T, N, Hkv, new):
    code, error, need = _call(T, N, Hkv, new, 0)
    assert (code, need > 0) == (-3, True) and b"workspace" in error, (code, error, need)
