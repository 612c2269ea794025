"""The paged cache and the attention over it on the GPU against the 64-bit oracle.

Tolerances, per value of the attention's output: half a step of bf16 (2^-8) of the value for the output's own rounding; the same of the weighted mean of |v| for the probabilities'
(each is off by 2^-8 of itself at most); and the mean of |v| times 4 ds, where ds bounds a logit's error in 32 bits: (D + 8) 2^-24 times the scaled sum of |q||k|, the largest of the
row (a weight is off by 2 ds of itself through its own and the row's sum's logits, and as much is left for the exponentials, off by 2^-22, and the sums).  lse: 2 ds + 2^-18."""
import math

import pytest
import torch

import vlm_training_amd as V
from oracle import cache_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, E4 = torch.bfloat16, torch.float8_e4m3fn


def _offsets(parts):
    return torch.tensor([sum(parts[:i]) for i in range(len(parts) + 1)], dtype=torch.int32)


def make(kind, lens, hkv, dim, page, seed=0, spare=2, std=1.0, width=None):
    """Requests' keys and values (a list of (L, hkv, dim) pairs, bf16 on the CPU) and the cache that holds them, on the GPU, with pages in a random order and noise where nothing is."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in lens]
    pages = sum(need) + spare
    order, at = torch.randperm(pages, generator=g).int(), 0
    table = torch.full((len(lens), width or max(max(need), 1)), -1, dtype=torch.int32)
    cache = V.KvCache.empty(pages, hkv, dim, page=page, dtype=BF if kind == "bf16" else E4, device="cpu")
    for pool in (cache.k, cache.v):
        if kind == "bf16":
            pool.copy_(torch.randn(pool.shape, generator=g) * 3)
        else:
            pool.view(torch.uint8).copy_(torch.randint(0, 256, pool.shape, generator=g))
    rows = []
    for i, n in enumerate(lens):
        table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
        k, v = ((torch.randn(n, hkv, dim, generator=g) * std).to(BF) for _ in range(2))
        rows.append([k, v])
        for pool, scale, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
            if n and kind == "e4m3":
                y, e = R.quantise(x)
                codes, powers = y.float().to(E4).view(torch.uint8), (e + 127).to(torch.uint8)
            for b in range(need[i]):
                id, part = int(table[i, b]), slice(b * page, min(n, (b + 1) * page))
                if kind == "bf16":
                    pool[id, :, :part.stop - part.start] = x[part].transpose(0, 1)
                else:
                    pool.view(torch.uint8)[id, :, :part.stop - part.start] = codes[part].transpose(0, 1)
                    scale.view(torch.uint8)[id, :, :part.stop - part.start] = powers[part].transpose(0, 1)
    return rows, V.KvCache(*(t if t is None else t.to(DEV) for t in cache._parts())), table.to(DEV)


def put(cache, table, i, p, k, v):
    """Row p of request i into a cache on the CPU, as the oracle rounds it."""
    page = cache.k.shape[2]
    at = (int(table[i, p // page]), slice(None), p % page)
    for pool, scale, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
        if scale is None:
            pool[at] = x
        else:
            y, e = R.quantise(x)
            pool.view(torch.uint8)[at] = y.float().to(E4).view(torch.uint8)
            scale.view(torch.uint8)[at] = torch.where(torch.isfinite(y).all(-1), e + 127, 255).to(torch.uint8)


def check(out, lse, q, rows, kind, new, lens, scale):
    at = 0
    for (k, v), m, n in zip(rows, new, lens):
        x = q[at:at + m].cpu()
        k, v = R.stored(k, kind), R.stored(v, kind)
        limits = [n - m + i for i in range(m)]
        want, want_lse = R.attend(x, k, v, scale, limits)
        mean, _ = R.attend(x, k, v.abs(), scale, limits)
        group = x.shape[1] // k.shape[1]
        sums = abs(scale) * torch.einsum("ihd,lhd->hil", x.double().abs(), k.abs().repeat_interleave(group, 1)) if n else torch.zeros(x.shape[1], m, 1, dtype=torch.float64)
        live = torch.arange(sums.shape[2])[None] <= torch.tensor(limits)[:, None]
        ds = (x.shape[2] + 8) * 2.0 ** -24 * (sums * live).amax(-1)                       # (heads, rows)
        bound = 2.0 ** -8 * (want.abs() + mean) + 4 * ds.T[..., None] * mean
        got = out[at:at + m].cpu().double()
        assert torch.isfinite(got).all()
        worst = ((got - want).abs() - bound).max().item() if m else 0
        assert worst <= 0, f"over its bound by {worst:.3g}, largest error {(got - want).abs().max():.3g}"
        if lse is not None and m:
            mine = lse[:, at:at + m].cpu().double()
            none = want_lse == -math.inf
            assert torch.equal(mine == -math.inf, none)
            assert ((mine - want_lse).abs() <= 2 * ds + 2.0 ** -18)[~none].all()
        at += m
    assert (out[at:] == 0).all() and (lse is None or (lse[:, at:] == -math.inf).all())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (256, 32)])
def test_walks_over_many_pages(kind, dim, page):
    """Several hundred pages to a walk; blocks in pieces; chunks that end in the middle of a block."""
    print(kind, dim, page, flush=True)
    new, lens = [75, 1, 40], [6500, 5300, 40]
    rows, cache, table = make(kind, lens, 1, dim, page, seed=9)
    q = (torch.randn(sum(new), 4, dim, generator=torch.Generator().manual_seed(1)) * 1.5).to(BF).to(DEV)
    cu, lengths = _offsets(new).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    for some in (slice(0, 3), slice(0, 1)):
        n = sum(new[some])
        out, lse = V.paged_attn(q[:n], cache, table[some], cu[:len(new[some]) + 1], lengths[some], return_lse=True)
        check(out, lse, q[:n], rows[some], kind, new[some], lens[some], dim ** -0.5)


GEOMETRY = [(4, 4, 64, 16), (8, 2, 128, 64), (6, 3, 72, 32), (16, 1, 128, 128), (5, 1, 80, 16), (4, 2, 256, 64), (3, 1, 96, 256), (2, 1, 8, 16), (12, 2, 144, 64)]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("hq,hkv,dim,page", GEOMETRY)
@pytest.mark.parametrize("shape", ["one", "steps", "drafts", "chunks"])
def test_attention(kind, hq, hkv, dim, page, shape):
    if kind == "e4m3" and dim % 16:
        pytest.skip("8-bit rows are multiples of 16")
    print(shape, kind, hq, hkv, dim, page, flush=True)
    new, lens = {"one": ([1], [1]), "steps": ([1] * 7, [1, 31, 32, 33, 65, 300, 17]), "drafts": ([3, 0, 2, 8, 1], [3, 40, 257, 64, 16]),
                 "chunks": ([70, 1, 0, 129, 5, 33], [70, 100, 0, 333, 5, 290])}[shape]
    rows, cache, table = make(kind, lens, hkv, dim, page, seed=dim)
    g = torch.Generator().manual_seed(7)
    q = (torch.randn(sum(new) + 3, hq, dim, generator=g) * 1.5).to(BF).to(DEV)
    cu, lengths = _offsets(new).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    out, lse = V.paged_attn(q, cache, table, cu, lengths, return_lse=True)
    check(out, lse, q, rows, kind, new, lens, dim ** -0.5)
    # (bounds that are known change which kernels run)
    out, lse = V.paged_attn(q, cache, table, cu.long(), lengths.long(), max_new=max(new), max_length=max(lens), return_lse=True)
    check(out, lse, q, rows, kind, new, lens, dim ** -0.5)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("hkv,dim,page", [(1, 16, 16), (3, 72, 32), (8, 128, 64), (2, 256, 128), (5, 80, 256), (16, 64, 16)])
def test_write_and_read(kind, hkv, dim, page):
    if kind == "e4m3" and dim % 16:
        pytest.skip("8-bit rows are multiples of 16")
    print(kind, hkv, dim, page, flush=True)
    new, lens = [0, 1, 70, 3, 0, 33, 5], [4, 1, 200, 64, 0, 33, 300]
    rows, cache, table = make(kind, lens, hkv, dim, page, seed=3)
    want = V.KvCache(*(t if t is None else t.cpu() for t in cache._parts()))
    g = torch.Generator().manual_seed(11)
    total = sum(new)
    wide = torch.randn(total + 4, 3 * hkv, dim, generator=g) * torch.logspace(-4, 4, 3 * hkv)[:, None]
    wide[2, :, 1:] = 0
    wide[5] = 0
    wide = wide.to(BF)
    k, v = wide[:, hkv:2 * hkv], wide[:, 2 * hkv:]
    at = 0
    for i, (m, n) in enumerate(zip(new, lens)):
        for j in range(m):
            put(want, table.cpu(), i, n - m + j, k[at + j], v[at + j])
        at += m
    dev = wide.to(DEV)
    cu, lengths = _offsets(new).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    versions = [t._version for t in cache._parts() if t is not None]
    V.kv_cache_write(cache, dev[:, hkv:2 * hkv], dev[:, 2 * hkv:], table, cu, lengths)
    assert all(t._version > n for t, n in zip((t for t in cache._parts() if t is not None), versions))
    for got, ref in zip(cache._parts(), want._parts()):
        if got is not None:
            assert torch.equal(got.cpu().view(torch.uint8), ref.view(torch.uint8))         # the rows written, and everything else as it was
    # the rows just written, and all rows of each request
    back = V.kv_cache_read(cache, table, cu, total + 2, first=torch.tensor([n - m for n, m in zip(lens, new)], device=DEV))
    for got, x in zip(back, (k, v)):
        assert torch.equal(got[:total].cpu().double(), R.stored(x[:total], kind)) and (got[total:] == 0).all()
    back = V.kv_cache_read(cache, table, _offsets(lens).to(DEV), sum(lens))
    at = 0
    for i, n in enumerate(lens):
        for got, x, fresh in zip(back, rows[i], (k, v)):
            start = sum(new[:i])
            old = R.stored(x[:n - new[i]], kind)
            assert torch.equal(got[at:at + n - new[i]].cpu().double(), old)
            assert torch.equal(got[at + n - new[i]:at + n].cpu().double(), R.stored(fresh[start:start + new[i]], kind))
        at += n


def test_every_stored_value_is_read_exactly():
    """All e4m3 values under every power that is written; NaN is NaN."""
    page, dim = 256, 256
    cache = V.KvCache.empty(1, 1, dim, page=page, dtype=E4)
    codes = torch.arange(256, dtype=torch.uint8).expand(page, dim)
    cache.k.view(torch.uint8)[0, 0] = codes.to(DEV)
    cache.k_scale.view(torch.uint8)[0, 0] = torch.arange(256, dtype=torch.uint8, device=DEV)
    got, _ = V.kv_cache_read(cache, torch.zeros(1, 1, dtype=torch.int32, device=DEV), _offsets([page]).to(DEV), page)
    got = got[:, 0].cpu().double()
    value = codes.view(E4).double() * torch.exp2(torch.arange(256, dtype=torch.float64) - 127)[:, None]
    nan = torch.isnan(codes.view(E4).double())
    assert torch.isnan(got[nan]).all()
    assert torch.isnan(got[255]).all()
    for byte in range(27, 247):
        assert torch.equal(got[byte][~nan[byte]], value[byte][~nan[byte]]), byte


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_rows_that_are_not_finite_are_stored_as_such(kind):
    cache = V.KvCache.empty(1, 2, 64, page=16, dtype=BF if kind == "bf16" else E4)
    x = torch.ones(3, 2, 64, dtype=BF)
    x[0, 0, 5], x[1, 1, 63], x[2, 0, 0] = math.inf, math.nan, -math.inf
    table, cu = torch.zeros(1, 1, dtype=torch.int32, device=DEV), _offsets([3]).to(DEV)
    V.kv_cache_write(cache, x.to(DEV), x.to(DEV), table, cu, torch.tensor([3], device=DEV))
    for got in V.kv_cache_read(cache, table, cu, 3):
        assert torch.equal(got.cpu().double().nan_to_num(7, 8, 9), R.stored(x, kind).nan_to_num(7, 8, 9))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dim,m", [(128, 4), (64, 40), (256, 13)])
def test_what_is_not_attended_never_reaches_a_row(kind, page, dim, m):
    """Infinities and NaN in later tokens of the chunk, behind the request's end and on other requests' pages."""
    new, lens, hkv, hq = [m, 1, m], [90 + m, 33, m], 2, 4
    rows, cache, table = make(kind, lens, hkv, dim, page)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(sum(new), hq, dim, generator=g).to(BF).to(DEV)
    cu, lengths = _offsets(new).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    bad = m // 2
    def poison(i, p, head, value):
        id, place = int(table[i, p // page]), p % page
        for pool in (cache.k, cache.v):
            if kind == "bf16":
                pool[id, head, place, 3::7] = value
            else:
                pool.view(torch.uint8)[id, head, place] = 0x7f
    for i in (0, 2):
        poison(i, lens[i] - m + bad, 1, math.nan)
        poison(i, lens[i] - 1, 0, math.inf)
        for x in rows[i]:
            x[lens[i] - m + bad, 1] = 0               # (what the rows in front of it see does not depend on it)
            x[lens[i] - 1, 0] = 0
    for i, n in enumerate(lens):
        for p in range(n, (n + page - 1) // page * page):
            poison(i, p, 0, math.nan)
            poison(i, p, 1, -math.inf)
    out, lse = V.paged_attn(q, cache, table, cu, lengths, return_lse=True)
    out, lse, q = out.cpu(), lse.cpu(), q.cpu()
    at = 0
    for i, (n_new, n) in enumerate(zip(new, lens)):
        clean = [bad if i != 1 else 1, n_new - 1 if i != 1 else 1]       # rows that see nothing of it: of kv head 1, of kv head 0
        for heads, kv, rows_clean in ((slice(2, 4), 1, clean[0]), (slice(0, 2), 0, clean[1])):
            part = [[x[:n - n_new + rows_clean, kv:kv + 1] for x in rows[i]]]
            check(out[at:at + rows_clean, heads].contiguous(), lse[heads, at:at + rows_clean].contiguous(), q[at:at + rows_clean, heads], part, kind, [rows_clean],
                  [n - n_new + rows_clean], dim ** -0.5)
            if i != 1:
                assert torch.isnan(out[at + rows_clean:at + n_new, heads]).all(dim=-1).any(dim=-1).all()
        at += n_new


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_places_that_are_nowhere(kind):
    """Pages outside the pool, positions outside the table or in front of the request: not written, zeros, zero keys and values."""
    page, hkv, dim, lens = 16, 2, 64, [40, 70, 3]
    rows, cache, table = make(kind, lens, hkv, dim, page)
    table[0, 1], table[1, 2] = 1 << 30, -5
    before = [None if t is None else t.clone() for t in cache._parts()]
    x = torch.ones(12, hkv, dim, dtype=BF, device=DEV)
    # request 0: positions 28 .. 33, of which 28 .. 31 lie on the page that is none; 1: behind its table; 2: three rows in front of its first
    new = [6, 2, 4]
    V.kv_cache_write(cache, x, x, table, _offsets(new).to(DEV), torch.tensor([34, 90, 1], device=DEV))
    changed = [(a.view(torch.uint8) != b.view(torch.uint8)).flatten(3).any(-1) for a, b in ((cache.k, before[0]), (cache.v, before[1]))]
    assert all(c.any(1).sum() == 3 for c in changed)          # positions 32, 33 of request 0, position 0 of request 2
    for t, b in zip(cache._parts(), before):
        if t is not None:
            t.view(torch.uint8).copy_(b.view(torch.uint8))
    read = V.kv_cache_read(cache, table, _offsets([40, 90, 3]).to(DEV), 133)
    for k in range(2):
        rows[0][k][16:32] = 0
        rows[1][k][32:48] = 0
        at = 0
        for i, n in enumerate((40, 70, 3)):
            assert torch.equal(read[k][at:at + n].cpu().double(), R.stored(rows[i][k], kind))
            at += n if i != 1 else 90
        assert (read[k][40 + 80:40 + 90] == 0).all()
    back = V.kv_cache_read(cache, table, _offsets([3, 0, 0]).to(DEV), 3, first=torch.tensor([-2, 0, 0], device=DEV))
    assert (back[0][:2] == 0).all() and torch.equal(back[0][2].cpu().double(), R.stored(rows[0][0][0], kind))
    q = torch.randn(9, 4, dim, generator=torch.Generator().manual_seed(2)).to(BF).to(DEV)
    new = [3, 1, 5]                                           # (request 2 is shorter than its new rows: two of them have no key)
    out, lse = V.paged_attn(q, cache, table, _offsets(new).to(DEV), torch.tensor(lens, device=DEV), return_lse=True)
    check(out, lse, q, rows, kind, new, lens, dim ** -0.5)
    assert (out[4:6] == 0).all()
    # lengths beyond the table: the keys end with it
    full = table.shape[1] * page
    out = V.paged_attn(q[:1], cache, table[2:], _offsets([1]).to(DEV), torch.tensor([full + 1000], device=DEV))
    k, v = (torch.zeros(full, hkv, dim, dtype=BF) for _ in range(2))
    got = V.kv_cache_read(cache, table[2:], _offsets([full]).to(DEV), full)
    want, _ = R.attend(q[:1].cpu(), got[0].cpu(), got[1].cpu(), dim ** -0.5, [full - 1])
    none = torch.isnan(want)                                  # (the 8-bit noise behind the request's rows holds NaN)
    assert torch.equal(torch.isnan(out.cpu()), none) and (kind == "e4m3" or not none.any())
    most = got[1].cpu().double().nan_to_num(0).abs().max().item()      # (2^-8 of the value and of the mean of |v|, and what the logits' rounding leaves: 4 ds is below 2^-10)
    worst = (out.cpu().double() - want).abs()[~none].max().item() if not none.all() else 0.0
    assert worst <= 2.0 ** -7 * max(1.0, most)


def test_scales():
    """Softmax scales that are negative, zero, large; logits far apart."""
    lens, new = [200, 50], [2, 20]
    rows, cache, table = make("bf16", lens, 2, 64, 32)
    q = torch.randn(sum(new), 4, 64, generator=torch.Generator().manual_seed(3)).to(BF).to(DEV)
    cu, lengths = _offsets(new).to(DEV), torch.tensor(lens, device=DEV)
    for scale in (-0.2, 0.0, 3.0, 1e-30):
        out, lse = V.paged_attn(q, cache, table, cu, lengths, softmax_scale=scale, return_lse=True)
        check(out, lse, q, rows, "bf16", new, lens, scale)


def test_views():
    """q, k, v as slices of wider tensors, on no 16-byte boundary too; pools that are slices of one for all layers; a table that is a slice."""
    page, hkv, hq, dim, lens, new = 32, 2, 4, 64, [40, 100], [3, 5]
    rows, cache, table = make("bf16", lens, hkv, dim, page, width=6)
    pool = torch.zeros(cache.k.shape[0], 3, 2, *cache.k.shape[1:], dtype=BF, device=DEV)
    pool[:, 1, 0], pool[:, 1, 1] = cache.k, cache.v
    view = V.KvCache(pool[:, 1, 0], pool[:, 1, 1])
    cu, lengths = _offsets(new).to(DEV), torch.tensor(lens, device=DEV)
    wide = torch.randn(sum(new), hq + 2, dim + 9, generator=torch.Generator().manual_seed(4)).to(BF).to(DEV)
    q = wide[:, 1:1 + hq, 3:3 + dim]
    out, lse = V.paged_attn(q, view, table[:, :4], cu, lengths, return_lse=True)
    check(out, lse, q, rows, "bf16", new, lens, dim ** -0.5)
    flat = torch.randn(sum(new), hq * dim, generator=torch.Generator().manual_seed(4)).to(BF).to(DEV)
    q = flat.view(sum(new), dim, hq).transpose(1, 2)
    check(*V.paged_attn(q, view, table, cu, lengths, return_lse=True), q, rows, "bf16", new, lens, dim ** -0.5)
    k = wide[:, 2:2 + hkv, 1:1 + dim]
    V.kv_cache_write(view, k, k, table, cu, lengths)
    back = V.kv_cache_read(view, table, cu, sum(new), first=lengths - torch.tensor(new, device=DEV))
    assert torch.equal(back[0], k) and torch.equal(back[1], k) and (pool[:, 0] == 0).all() and (pool[:, 2] == 0).all()


def test_refusals():
    lens, new = [20, 5], [2, 3]
    rows, cache, table = make("bf16", lens, 2, 64, 16)
    _, small, _ = make("e4m3", lens, 2, 64, 16)
    q = torch.zeros(5, 4, 64, dtype=BF, device=DEV)
    k = torch.zeros(5, 2, 64, dtype=BF, device=DEV)
    cu, lengths = _offsets(new).to(DEV), torch.tensor(lens, device=DEV)
    ok = dict(q=q, cache=cache, table=table, cu=cu, lengths=lengths, k=k, v=k)

    def attn(**c):
        c = {**ok, **c}
        return V.paged_attn(c["q"], c["cache"], c["table"], c["cu"], c["lengths"], **{n: c[n] for n in ("max_new", "max_length", "softmax_scale") if n in c})

    def write(**c):
        c = {**ok, **c}
        return V.kv_cache_write(c["cache"], c["k"], c["v"], c["table"], c["cu"], c["lengths"])

    def read(**c):
        c = {**ok, **c}
        return V.kv_cache_read(c["cache"], c["table"], c["cu"], c.get("rows", 5), first=c.get("first"))

    attn(), write(), read()
    half = [dict(cache=V.KvCache(cache.k.half(), cache.v.half())), dict(cache=V.KvCache(cache.k, cache.v[:, :1])), dict(cache=V.KvCache(cache.k, small.v)),
            dict(cache=V.KvCache(cache.k, cache.v, small.k_scale, small.v_scale)), dict(cache=V.KvCache(small.k, small.v)), dict(cache=V.KvCache(small.k, small.v, small.k_scale, small.v_scale[:1])),
            dict(cache=V.KvCache(cache.k.transpose(1, 2), cache.v.transpose(1, 2))), dict(cache=V.KvCache(cache.k[..., ::2], cache.v[..., ::2])), dict(table=table[:1]), dict(table=table.float()),
            dict(table=table[0]), dict(cu=cu[:2]), dict(cache=V.KvCache(cache.k[:, :, :8], cache.v[:, :, :8])), dict(cache=V.KvCache(cache.k.view(-1)[4:4 + 1024].view(1, 1, 16, 64), cache.v[:1, :1]))]
    for change in half:
        for call in (attn, write, read):
            with pytest.raises((ValueError, RuntimeError)):
                call(**change)
    for change in (dict(q=q.float()), dict(q=q[..., :32]), dict(q=q[:, :3]), dict(q=q[0]), dict(lengths=lengths[:1]), dict(lengths=lengths.float()), dict(max_new=0), dict(max_length=0),
                   dict(softmax_scale=math.inf), dict(q=q.clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            attn(**change)
    for change in (dict(k=k.float()), dict(v=k[:, :1]), dict(v=k[:4]), dict(k=k[..., :32]), dict(lengths=lengths[:1]), dict(k=k.clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            write(**change)
    for change in (dict(rows=-1), dict(first=lengths[:1])):
        with pytest.raises(ValueError):
            read(**change)
    with pytest.raises(RuntimeError, match="GPU only"):
        attn(lengths=lengths.cpu())
    with pytest.raises(ValueError):
        V.paged_attn(torch.zeros(5, 34, 64, dtype=BF, device=DEV)[:, :33], V.KvCache.empty(2, 2, 64), table, cu, lengths)
    empty = V.paged_attn(q[:0], cache, table, torch.zeros_like(cu), lengths)
    assert empty.shape == (0, 4, 64)
    V.kv_cache_write(cache, k[:0], k[:0], table, torch.zeros_like(cu), lengths)
    assert V.kv_cache_read(cache, table, torch.zeros_like(cu), 0)[0].shape == (0, 2, 64)
