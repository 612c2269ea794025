"""Paged attention where a request's length passes what its table holds: the keys end with the table, and every one of them counts.

The cache is full of finite noise, so that every output is a number; tolerances as in test_gpu_cache.py."""
import pytest
import torch

import vlm_training_amd as V
from tests.test_gpu_cache import BF, DEV, E4, _offsets
from tests.test_gpu_cache_pages import compare

pytestmark = pytest.mark.gpu


def _noise(kind, pages, hkv, dim, page):
    g = torch.Generator().manual_seed(dim)
    if kind == "bf16":
        return V.KvCache(*(torch.randn(pages, hkv, page, dim, generator=g).to(BF).to(DEV) for _ in range(2)))
    codes = [torch.randint(0, 256, (pages, hkv, page, dim), generator=g).to(torch.uint8) for _ in range(2)]
    codes = [torch.where((c & 0x7f) == 0x7f, c ^ 1, c).to(DEV).view(E4) for c in codes]           # (no NaN)
    return V.KvCache(*codes, *(torch.randint(117, 121, (pages, hkv, page), generator=g).to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu) for _ in range(2)))


# new rows and, for each request, by how much its length passes the table (negative: it does not)
SHAPES = [([1], [1000]), ([1, 1], [3, -5]), ([4, 1, 2], [2, 0, 10]), ([70], [1000]), ([70, 1, 40], [30, 7, -11])]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (256, 64)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("width", [3, 40])
def test_keys_end_with_the_table(kind, dim, page, shape, width):
    new, past = SHAPES[shape]
    print(kind, dim, page, new, past, width, flush=True)
    hkv, hq, full, n = 2, 8, width * page, len(new)
    cache = _noise(kind, n * width + 3, hkv, dim, page)
    table = torch.randperm(n * width + 3, generator=torch.Generator().manual_seed(1))[:n * width].int().view(n, width).to(DEV)
    k, v = (x.split(full) for x in V.kv_cache_read(cache, table, _offsets([full] * n).to(DEV), n * full))
    assert all(torch.isfinite(x).all() for x in k + v)
    q = (torch.randn(sum(new), hq, dim, generator=torch.Generator().manual_seed(2)) * 0.5).to(BF).to(DEV)
    lens = [full + p for p in past]
    out, lse = V.paged_attn(q, cache, table, _offsets(new).to(DEV), torch.tensor(lens, device=DEV), return_lse=True)
    at = 0
    for i, m in enumerate(new):
        for j in range(m):
            keys = min(lens[i] - m + j + 1, full)
            row = slice(at + j, at + j + 1)
            if keys <= 0:                                 # (a row in front of its request's first key)
                assert (out[row] == 0).all() and (lse[:, row] == -torch.inf).all()
                continue
            compare(out[row], lse[:, row], q[row], k[i][:keys], v[i][:keys], keys, dim ** -0.5)
        at += m
