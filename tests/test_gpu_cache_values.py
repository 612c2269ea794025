"""The paged cache at the ends of what values and integers can be: NaN that a row does attend, rows next to bf16's largest value, numbers past 32 bits."""
import math

import pytest
import torch

import vlm_training_amd as V
from oracle import cache_ref as R
from tests.test_gpu_cache import BF, DEV, E4, _offsets, check, make

pytestmark = pytest.mark.gpu


def _place(cache, table, i, p):
    page = cache.k.shape[2]
    return int(table[i, p // page]), slice(None), p % page


# (new rows, lengths, (request, position) of the NaN key): alone in its tile, a row's only key, first, in the middle of a long request, in a chunk
CASES = [([1, 1], [33, 700], [(0, 32), (1, 0)]), ([1, 2], [1, 65], [(0, 0), (1, 63)]), ([1], [20000], [(0, 9000)]), ([60], [60], [(0, 0)]), ([60, 1, 40], [97, 400, 3000], [(0, 96), (2, 2990)]),
         ([200], [9000], [(0, 8999)])]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("width", [None, 1200])
def test_nan_that_is_attended_shows(kind, dim, case, width):
    """A NaN key makes every row that attends it NaN, a NaN query its own row; all others are as they were."""
    new, lens, where = CASES[case]
    hkv, hq = 2, 6
    print(kind, dim, new, lens, width, flush=True)
    rows, cache, table = make(kind, lens, hkv, dim, 64, seed=3, width=width)
    q = torch.randn(sum(new), hq, dim, generator=torch.Generator().manual_seed(4)).to(BF).to(DEV)
    cu, lengths = _offsets(new).to(DEV), torch.tensor(lens, device=DEV)
    clean = V.paged_attn(q, cache, table, cu, lengths, return_lse=True)
    check(*clean, q, rows, kind, new, lens, dim ** -0.5)

    def compare(out, lse, bad):                              # bad (rows, heads)
        assert torch.isnan(out[bad]).all() and torch.isnan(lse.T[bad]).all()
        check(torch.where(bad[..., None], clean[0], out), torch.where(bad.T, clean[1], lse), q, rows, kind, new, lens, dim ** -0.5)

    bad = torch.zeros(sum(new), hq, dtype=torch.bool, device=DEV)
    bad[0, 1] = bad[-1, 4] = True
    x = q.clone()
    x[bad] = math.nan
    compare(*V.paged_attn(x, cache, table, cu, lengths, return_lse=True), bad)
    bad = torch.zeros_like(bad)
    for i, p in where:
        if kind == "bf16":
            cache.k[_place(cache, table, i, p)][1] = math.nan
        else:
            cache.k.view(torch.uint8)[_place(cache, table, i, p)][1] = 0x7f
        at = sum(new[:i])
        bad[at + max(0, p - (lens[i] - new[i])):at + new[i], hq // 2:] = True
    compare(*V.paged_attn(q, cache, table, cu, lengths, return_lse=True), bad)


@pytest.mark.parametrize("new,length,width", [(1, 20000, None), (60, 20000, None), (3, 40, None), (60, 300, 1200)])
def test_nan_shows_beside_logits_far_above_it(new, length, width):
    """One key's logits are some 10 000 above all others: the other pieces' weights are 0 in 32 bits, a NaN among them is not."""
    for far, nan in ((0, length // 2), (length - new, 3)):
        rows, cache, table = make("bf16", [length], 1, 64, 64, seed=3, width=width)
        q = torch.rand(new, 4, 64, generator=torch.Generator().manual_seed(4)).to(BF).to(DEV) + 1
        cache.k[_place(cache, table, 0, far)] = 1000.0
        cache.k[_place(cache, table, 0, nan)] = math.nan
        out, lse = V.paged_attn(q, cache, table, _offsets([new]).to(DEV), torch.tensor([length], device=DEV), return_lse=True)
        seen = torch.arange(length - new, length, device=DEV) >= nan
        assert torch.isnan(out[seen]).all() and torch.isnan(lse[:, seen]).all() and torch.isfinite(out[~seen]).all()


def test_rows_next_to_the_largest_value():
    """8-bit rows whose largest value lies within one rounding of 2^128: 240 powers of two, never an infinity, by at most 2^-4 of the value."""
    big = torch.tensor([0x7f60, 0x7f61, 0x7f70, 0x7f77, 0x7f78, 0x7f79, 0x7f7f], dtype=torch.int16).view(BF)
    x = torch.zeros(2 * len(big), 2, 64, dtype=BF)
    for i, b in enumerate(big):
        x[2 * i, 0, 3], x[2 * i, 0, 60], x[2 * i, 1, 0] = b, -b, 1.0
        x[2 * i + 1, 1] = -b
    cache = V.KvCache.empty(1, 2, 64, page=16, dtype=E4)
    table, cu = torch.zeros(1, 1, dtype=torch.int32, device=DEV), _offsets([len(x)]).to(DEV)
    V.kv_cache_write(cache, x.to(DEV), -x.to(DEV), table, cu, torch.tensor([len(x)], device=DEV))
    k, v = (t.cpu().double() for t in V.kv_cache_read(cache, table, cu, len(x)))
    assert torch.equal(k, R.stored(x, "e4m3")) and torch.equal(v, -k) and torch.isfinite(k).all()
    assert ((k - x.double()).abs() <= 2.0 ** -4 * x.double().abs()).all()


def test_numbers_past_32_bits():
    """int64 page numbers and lengths that no int32 holds are what they say - nowhere, beyond the table -, not their low halves."""
    lens, dim = [40, 40], 64
    rows, cache, table = make("bf16", lens, 2, dim, 16)
    far = table.long()
    far[0, 1] += 1 << 32
    far[1, 0] -= 1 << 33
    cu = _offsets([1, 1]).to(DEV)
    gone = table.clone()
    gone[0, 1] = gone[1, 0] = -1
    q = torch.randn(2, 4, dim, generator=torch.Generator().manual_seed(4)).to(BF).to(DEV)
    lengths = torch.tensor(lens, device=DEV)
    assert torch.equal(V.paged_attn(q, cache, far, cu, lengths), V.paged_attn(q, cache, gone, cu, lengths))
    before = cache.k.clone()
    for length in ((1 << 32) + 40, -(1 << 32) + 40, (1 << 31) - 1, -(1 << 31)):
        V.kv_cache_write(cache, q[:, :2], q[:, :2], table, cu, torch.tensor([length] * 2, device=DEV))
        assert torch.equal(cache.k, before), length
    got = V.paged_attn(q, cache, table, cu, torch.tensor([-(1 << 32) + 40] * 2, device=DEV))
    assert (got == 0).all()
    back = V.kv_cache_read(cache, table, _offsets([8, 8]).to(DEV), 16, first=torch.tensor([1 << 32, -(1 << 32)], device=DEV))
    assert (back[0] == 0).all() and (back[1] == 0).all()
