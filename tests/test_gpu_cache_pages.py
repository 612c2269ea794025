"""Chunks over long caches on small pages: walks whose pieces begin anywhere among a request's pages, against attention in 64 bits.

The lengths are such that some block's pieces begin one or two tiles in front of a page whose number in the table is a multiple of 64, and go on past the next such page.
Tolerances as in test_gpu_cache.py."""
import math

import pytest
import torch

import vlm_training_amd as V
from tests.test_gpu_cache import BF, DEV, E4, _offsets

pytestmark = pytest.mark.gpu


def filled(kind, lens, hkv, dim, page, seed):
    """A cache with requests of random rows on pages in a random order, its table, and the rows as it holds them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    order = torch.randperm(sum(need) + 5, generator=g, device=DEV).int()
    table, at = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEV), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    cache = V.KvCache.empty(len(order), hkv, dim, page=page, dtype=BF if kind == "bf16" else E4)
    k, v = (torch.randn(sum(lens), hkv, dim, generator=g, device=DEV).to(BF) for _ in range(2))
    cu, lengths = _offsets(lens).to(DEV), torch.tensor(lens, device=DEV)
    V.kv_cache_write(cache, k, v, table, cu, lengths)
    back = V.kv_cache_read(cache, table, cu, sum(lens))
    if kind == "bf16":
        assert torch.equal(back[0], k) and torch.equal(back[1], v)
    return cache, table, lengths, [x.split(lens) for x in back]


def compare(out, lse, q, k, v, length, scale):
    """One request: q (m, Hq, D), k, v (length, Hkv, D) bf16 on the GPU; products, statistics and sums in 64 bits."""
    m, hq, dim = q.shape
    group = hq // k.shape[1]
    live = torch.arange(length, device=DEV) <= torch.arange(length - m, length, device=DEV).repeat_interleave(group)[:, None]
    for h in range(k.shape[1]):
        mine = slice(h * group, (h + 1) * group)
        x, keys, values = q[:, mine].reshape(-1, dim).double(), k[:, h].double(), v[:, h].double()
        logits = (scale * (x @ keys.T.contiguous())).masked_fill(~live, -math.inf)
        weight = torch.softmax(logits, -1)
        want, mean = weight @ values, weight @ values.abs()
        ds = (dim + 8) * 2.0 ** -24 * (abs(scale) * (x.abs() @ keys.abs().T.contiguous())).masked_fill(~live, 0.0).amax(-1)
        got = out[:, mine].reshape(-1, dim).double()
        assert torch.isfinite(got).all()
        over = (got - want).abs() - (2.0 ** -8 * (want.abs() + mean) + 4 * ds[:, None] * mean)
        rows = (over > 0).any(-1).view(m, group).any(-1).nonzero().flatten().tolist()
        assert not rows, f"kv head {h}: {len(rows)} of {m} rows over their bound, {rows[0]} to {rows[-1]}, by up to {over.max():.3g}"
        gap = (lse[mine].T.reshape(-1).double() - torch.logsumexp(logits, -1)).abs()
        assert (gap <= 2 * ds + 2.0 ** -18).all()


# heads, kv heads, head_dim, page, new rows, lengths
CASES = [(16, 8, 64, 16, [579], [12081]), (16, 8, 64, 16, [586, 167, 1, 1], [8152, 5962, 1082, 405]), (16, 8, 64, 32, [585], [16243]),
         (16, 8, 64, 32, [591, 193, 1, 1], [12160, 12125, 578, 362]), (16, 8, 64, 64, [677], [34161]), (16, 8, 64, 64, [561, 25, 1, 1], [34780, 2046, 140, 439]),
         (32, 8, 128, 16, [512], [4492]), (32, 8, 128, 16, [300], [10300]), (32, 8, 128, 16, [640], [4417]), (32, 8, 128, 16, [408, 145, 1, 1], [6014, 1736, 382, 132]),
         (32, 8, 128, 32, [512], [9051]), (32, 8, 128, 32, [680], [8011]), (32, 8, 128, 32, [498, 124, 1, 1], [12181, 3361, 62, 137]), (32, 8, 128, 64, [512], [24474]),
         (32, 8, 128, 64, [680], [16896]), (32, 8, 128, 64, [592, 162, 1, 1], [16447, 280, 746, 364]), (16, 2, 256, 16, [509], [6033]),
         (16, 2, 256, 16, [483, 42, 1, 1], [6118, 42, 1527, 335]), (16, 2, 256, 32, [525], [12191]), (16, 2, 256, 32, [424, 25, 1, 1], [16273, 359, 381, 121]),
         (16, 2, 256, 64, [675], [16491]), (16, 2, 256, 64, [649, 141, 1, 1], [16477, 814, 1424, 474])]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_pieces_begin_anywhere_among_the_pages(kind, case):
    hq, hkv, dim, page, new, lens = CASES[case]
    print(kind, CASES[case], flush=True)
    cache, table, lengths, (k, v) = filled(kind, lens, hkv, dim, page, seed=case)
    q = (torch.randn(sum(new), hq, dim, generator=torch.Generator(device=DEV).manual_seed(case), device=DEV) * 1.5).to(BF)
    for kw in (dict(), dict(max_new=max(new), max_length=max(lens))):
        out, lse = V.paged_attn(q, cache, table, _offsets(new).to(DEV), lengths, return_lse=True, **kw)
        at = 0
        for i, (m, n) in enumerate(zip(new, lens)):
            compare(out[at:at + m], lse[:, at:at + m], q[at:at + m], k[i], v[i], n, dim ** -0.5)
            at += m
