"""Calls with so many rows that one for every four workgroups' lanes would pass 2^32 threads."""
import pytest
import torch

import vlm_training_amd as V
from tests.test_gpu_cache import BF, DEV, E4, _offsets

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,dim", [("bf16", 8), ("e4m3", 16)])
def test_more_than_two_to_the_26_rows(kind, dim):
    n, page = (1 << 26) + 773, 256
    print(kind, n, flush=True)
    pages = (n + page - 1) // page
    cache = V.KvCache.empty(pages, 1, dim, page=page, dtype=BF if kind == "bf16" else E4)
    table, cu, lengths = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=DEV)[None], _offsets([n]).to(DEV), torch.tensor([n], device=DEV)
    # (numbers that both kinds hold exactly: multiples of 1/8 up to 15/8)
    k = torch.randint(8, 16, (n, 1, dim), dtype=torch.int8, device=DEV).to(BF).div_(8)
    v = torch.randint(-15, -7, (n, 1, dim), dtype=torch.int8, device=DEV).to(BF).div_(8)
    V.kv_cache_write(cache, k, v, table, cu, lengths)
    back = V.kv_cache_read(cache, table, cu, n + 3)
    for got, x in zip(back, (k, v)):
        assert torch.equal(got[:n], x) and (got[n:] == 0).all()
