"""The paged cache as a serving loop uses it: captured steps, streams, many requests, shared pages, pools past 2^31 elements, long requests."""
import pytest
import torch

import vlm_training_amd as V
from oracle import cache_ref as R
from tests.test_gpu_cache import BF, DEV, E4, _offsets, check, make

pytestmark = pytest.mark.gpu


def _rand(shape, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(BF).to(DEV)


def _copy(cache):
    return V.KvCache(*(None if t is None else t.clone() for t in cache._parts()))


def _same(a, b):
    return all(x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a._parts(), b._parts()))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("new", [[1, 1, 1, 1, 1], [3, 1, 40, 0, 2]])
def test_a_captured_step_follows_its_lengths(kind, new):
    """One graph, replayed as the requests grow, with eager calls on another copy of the cache between the replays."""
    print(kind, new, flush=True)
    lens, hkv, hq, dim, page = [700, 1, 90, 33, 260], 2, 8, 128, 32
    rows, cache, table = make(kind, [n + 400 for n in lens], hkv, dim, page)
    other = _copy(cache)
    total = sum(new)
    cu, lengths = _offsets(new).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV) + 0
    q, k, v = _rand((total + 2, hq, dim), 1), _rand((total + 2, hkv, dim), 2), _rand((total + 2, hkv, dim), 3)

    def step(c, q, k, v, lengths):
        V.kv_cache_write(c, k, v, table, cu, lengths)
        out, lse = V.paged_attn(q, c, table, cu, lengths, max_new=max(new), return_lse=True)
        return (out, lse, *V.kv_cache_read(c, table, cu, total + 2, first=lengths - (cu[1:] - cu[:-1])))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(_copy(cache), q, k, v, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache, q, k, v, lengths)
    assert _same(cache, other)                            # (captured, not run)
    for turn in range(6):
        for t, n in ((q, 10), (k, 20), (v, 30)):
            t.copy_(_rand(t.shape, n + turn))
        lengths.add_(cu[1:] - cu[:-1])
        graph.replay()
        want = step(other, q.clone(), k.clone(), v.clone(), lengths.clone())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and _same(cache, other), turn


def test_calls_on_two_streams_at_once():
    """Each on a stream of its own, with a cache of its own, workspaces too; against the same calls one after the other."""
    lens = [3000, 1200, 5000]
    parts = [make(kind, lens, 2, 128, 64, seed=i) for i, kind in enumerate(("bf16", "e4m3"))]
    q = [_rand((3 + 50, 8, 128), i) for i in range(2)]
    cus, lengths = [_offsets(n).to(DEV) for n in ([1, 1, 1], [1, 50, 2])], torch.tensor(lens, device=DEV)
    want = [[V.paged_attn(q[i], parts[i][1], parts[i][2], cu, lengths) for cu in cus] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for turn in range(5):
        got = [[], []]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = [V.paged_attn(q[i], parts[i][1], parts[i][2], cu, lengths) for cu in cus]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_hundreds_of_requests(kind):
    """More requests than a wave has lanes, some without new rows, some with many: plans over several batches of them."""
    n = 333
    lens = [(i * 37) % 150 + (400 if i % 50 == 7 else 0) for i in range(n)]
    for new in ([min(1, k) if i % 5 else 0 for i, k in enumerate(lens)], [min(k, (0, 1, 2, 45, 1, 0, 7)[i % 7]) for i, k in enumerate(lens)]):
        rows, cache, table = make(kind, lens, 1, 64, 16, seed=1)
        q = _rand((sum(new) + 5, 2, 64), 4)
        cu, lengths = _offsets(new).to(DEV), torch.tensor(lens, device=DEV)
        out, lse = V.paged_attn(q, cache, table, cu, lengths, return_lse=True)
        check(out, lse, q, rows, kind, new, lens, 64 ** -0.5)
        again = V.paged_attn(q, cache, table, cu, lengths, max_new=max(new), max_length=max(lens))
        check(again, None, q, rows, kind, new, lens, 64 ** -0.5)
        k = _rand((sum(new) + 5, 1, 64), 5)
        V.kv_cache_write(cache, k, k, table, cu, lengths)
        back = V.kv_cache_read(cache, table, cu, sum(new), first=lengths - torch.tensor(new, device=DEV))
        assert torch.equal(back[0].cpu().double(), R.stored(k[:sum(new)].cpu(), kind)) and torch.equal(back[1], back[0])


def test_bounds_that_do_not_hold_cost_time_alone():
    lens, new = [900, 40, 2000], [60, 1, 33]
    rows, cache, table = make("bf16", lens, 2, 64, 32)
    q = _rand((sum(new), 4, 64), 1)
    cu, lengths = _offsets(new).to(DEV), torch.tensor(lens, device=DEV)
    for kw in (dict(max_new=1), dict(max_length=10), dict(max_new=5, max_length=33)):
        out, lse = V.paged_attn(q, cache, table, cu, lengths, return_lse=True, **kw)
        check(out, lse, q, rows, "bf16", new, lens, 64 ** -0.5)


def test_pages_that_requests_share():
    """A common prompt's pages in three tables, read by all; each goes on on pages of its own."""
    page, dim, hkv = 16, 64, 2
    rows, cache, table = make("bf16", [64, 20, 5, 33], hkv, dim, page, width=8)
    shared = torch.full((3, 8), -1, dtype=torch.int32)
    host = table.cpu()
    for i in range(3):
        shared[i, :4], shared[i, 4:7] = host[0, :4], host[i + 1, :3]
    lens, new = [84, 69, 97], [20, 1, 2]
    both = [[torch.cat([rows[0][x], rows[i + 1][x]]) for x in range(2)] for i in range(3)]
    q = _rand((sum(new), 4, dim), 2)
    out, lse = V.paged_attn(q, cache, shared.to(DEV), _offsets(new).to(DEV), torch.tensor(lens, device=DEV), return_lse=True)
    check(out, lse, q, both, "bf16", new, lens, dim ** -0.5)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_pools_past_two_to_the_31_elements(kind):
    """The last pages of a pool of 2.2e9 elements: written, read and attended where they lie."""
    pages, hkv, page, dim, n = 34000, 8, 64, 128, 150
    dtype = BF if kind == "bf16" else torch.uint8
    # (what no request holds is never written, so it may hold anything)
    pools = [torch.empty(pages, hkv, page, dim, dtype=dtype, device=DEV) for _ in range(2)]
    cache = V.KvCache(*pools) if kind == "bf16" else V.KvCache(*(p.view(E4) for p in pools), *(torch.empty(pages, hkv, page, dtype=torch.uint8, device=DEV) for _ in range(2)))
    assert pools[0].numel() > 2 ** 31
    table = torch.tensor([[pages - 1, 0, pages - 2], [pages - 3, pages // 2, pages - 4]], dtype=torch.int32, device=DEV)
    k, v = _rand((2 * n, hkv, dim), 1), _rand((2 * n, hkv, dim), 2)
    cu, lengths = _offsets([n, n]).to(DEV), torch.tensor([n, n], device=DEV)
    V.kv_cache_write(cache, k, v, table, cu, lengths)
    back = V.kv_cache_read(cache, table, cu, 2 * n)
    for got, x in zip(back, (k, v)):
        assert torch.equal(got.cpu().double(), R.stored(x.cpu(), kind))
    rows = [[x[:n].cpu() for x in (k, v)], [x[n:].cpu() for x in (k, v)]]
    for new in ([1, 1], [70, 3]):
        q = _rand((sum(new), 16, dim), 3)
        out, lse = V.paged_attn(q, cache, table, _offsets(new).to(DEV), lengths, return_lse=True)
        check(out, lse, q, rows, kind, new, [n, n], dim ** -0.5)


def test_a_request_of_300000_tokens():
    """One row and a chunk at the end of a long request, on pages of 16 in order; a row in its middle."""
    n, dim, page = 300007, 16, 16
    pages = (n + page - 1) // page
    k, v = _rand((n, 1, dim), 1), _rand((n, 1, dim), 2)
    cache, table = V.KvCache.empty(pages, 1, dim, page=page), torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    V.kv_cache_write(cache, k, v, table, _offsets([n]).to(DEV), torch.tensor([n], device=DEV))
    back = V.kv_cache_read(cache, table, _offsets([n]).to(DEV), n)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)
    kv = [[k.cpu(), v.cpu()]]
    for m, length in ((1, n), (40, n), (2, 150001)):
        q = _rand((m, 1, dim), 5, std=3.0)
        out, lse = V.paged_attn(q, cache, table, _offsets([m]).to(DEV), torch.tensor([length], device=DEV), return_lse=True)
        check(out, lse, q, [[x[:length] for x in kv[0]]], "bf16", [m], [length], dim ** -0.5)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [[1, 1, 1], [2, 5, 1], [60, 20, 1]])
def test_powers_behind_the_last_row_may_be_anything(dim, new):
    """Pages that were another request's before: NaN's power behind the last row, values that are NaN too."""
    lens = [70, 33, 1]
    rows, cache, table = make("e4m3", lens, 2, dim, 64, seed=2)
    for i, n in enumerate(lens):
        for p in range(n, (n + 63) // 64 * 64):
            for pool, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                scale.view(torch.uint8)[int(table[i, p // 64]), :, p % 64] = 255
                pool.view(torch.uint8)[int(table[i, p // 64]), :, p % 64, ::3] = 0x7f
    q = _rand((sum(new), 4, dim), 4)
    for kw in (dict(), dict(max_new=max(new), max_length=100)):
        out, lse = V.paged_attn(q, cache, table, _offsets(new).to(DEV), torch.tensor(lens, device=DEV), return_lse=True, **kw)
        check(out, lse, q, rows, "e4m3", new, lens, dim ** -0.5)


@pytest.mark.parametrize("hq,hkv", [(16, 1), (4, 2)])
def test_later_tokens_that_are_not_finite_with_a_bound_that_does_not_hold(hq, hkv):
    """One query to a block although there are three: a value behind it in its tile, infinite or NaN, stays out."""
    rows, cache, table = make("bf16", [40, 3], hkv, 64, 16)
    for i, n in ((0, 40), (1, 3)):
        page, place = int(table[i, (n - 1) // 16]), (n - 1) % 16
        cache.v[page, :, place] = float("nan")
        cache.v[page, 0, place, 0] = float("inf")
    q = _rand((6, hq, 64), 1)
    out, lse = V.paged_attn(q, cache, table, _offsets([3, 3]).to(DEV), torch.tensor([40, 3], device=DEV), max_new=1, return_lse=True)
    for at, i, n in ((0, 0, 40), (3, 1, 3)):
        check(out[at:at + 2], lse[:, at:at + 2], q[at:at + 2], [[x[:n - 1] for x in rows[i]]], "bf16", [2], [n - 1], 64 ** -0.5)
        assert not torch.isfinite(out[at + 2]).any()
