"""Calls without rows: there is nothing whose place in memory could matter.  Runs without a GPU (the pointers are never followed)."""
import pytest

from tests.test_cache_refusals import _args
from vlm_training_amd import _lib


@pytest.mark.parametrize("pointer,tok,head", [(16, 256, 73), (16, 3, 128), (22, 256, 128), (None, 0, 1)])
def test_views_without_rows_may_lie_anywhere(pointer, tok, head):
    lib = _lib.load()
    write = lambda T: lib.dsa_cache_write(_args(), pointer, tok, head, pointer, tok, head, 16, 16, T, 2, None)  # noqa: E731
    attn = lambda T: lib.dsa_paged_attn(_args(), pointer, tok, head, 16, 16, T, 2, 4, 1.0, 0, 0, 16, None, 16, 1 << 40, None)  # noqa: E731
    assert write(0) == 0 and attn(0) == 0, lib.dsa_last_error()
    assert write(8) == -1 and attn(8) == -1
