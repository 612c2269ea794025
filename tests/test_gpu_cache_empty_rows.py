"""Slices without rows of tensors in which no row lies on a 16-byte boundary: what such a slice with rows can do, one without can."""
import pytest
import torch

import vlm_training_amd as V
from tests.test_gpu_cache import BF, DEV, _offsets, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_slices_without_rows(kind):
    rows, cache, table = make(kind, [20, 5], 2, 64, 16)
    before = [None if t is None else t.clone() for t in cache._parts()]
    wide = torch.randn(7, 6, 73, device=DEV).to(BF)
    lengths = torch.tensor([20, 5], device=DEV)
    for m in (0, 2):
        cu = _offsets([m, 0]).to(DEV)
        q, k = wide[3:3 + m, 1:5, 5:69], wide[3:3 + m, 4:6, 3:67]
        out, lse = V.paged_attn(q, cache, table, cu, lengths, return_lse=True)
        assert out.shape == (m, 4, 64) and lse.shape == (4, m) and torch.isfinite(out).all()
        V.kv_cache_write(cache, k, k, table, cu, lengths)
        same = all(t is None or torch.equal(t.view(torch.uint8), b.view(torch.uint8)) for t, b in zip(cache._parts(), before))
        assert same == (m == 0)
