"""Operands of the paged cache at what its documentation says of them: rows that lie in the pools themselves, values as large as sums before the division have room for."""
import pytest
import torch

import vlm_training_amd as V
from tests.test_gpu_cache import BF, DEV, _offsets, make
from tests.test_gpu_cache_pages import compare

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128), (256, 72)])
def test_a_page_copied_to_another(page, dim):
    """A request that goes on by itself from a page that it shares: the rows come out of the pools that the call writes, from other pages."""
    _, cache, table = make("bf16", [2 * page, page + 5], 3, dim, page)
    before = cache.k.clone(), cache.v.clone()
    source, spare = int(table[1, 0]), sorted(set(range(cache.k.shape[0])) - set(table.flatten().tolist()))[0]
    k, v = (pool[source].transpose(0, 1) for pool in (cache.k, cache.v))
    V.kv_cache_write(cache, k, v, torch.tensor([[spare]], dtype=torch.int32, device=DEV), _offsets([page]).to(DEV), torch.tensor([page], device=DEV))
    for pool, old in zip((cache.k, cache.v), before):
        old[spare] = old[source]
        assert torch.equal(pool.view(torch.int16), old.view(torch.int16))


@pytest.mark.parametrize("new,length", [(1, 20000), (4, 500), (300, 9000)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_large_values(new, length, dim):
    """|v| up to 2^89: every sum of weights times values stays finite, whatever the number of keys."""
    print(new, length, dim, flush=True)
    rows, cache, table = make("bf16", [length], 2, dim, 64, seed=5)
    k, v = (x.to(DEV) for x in rows[0])
    v = (v.sign() * 2.0 ** 89).to(BF)
    V.kv_cache_write(cache, k, v, table, _offsets([length]).to(DEV), torch.tensor([length], device=DEV))
    q = torch.randn(new, 8, dim, generator=torch.Generator().manual_seed(1)).to(BF).to(DEV)
    out, lse = V.paged_attn(q, cache, table, _offsets([new]).to(DEV), torch.tensor([length], device=DEV), return_lse=True)
    compare(out, lse, q, k, v, length, dim ** -0.5)
