"""What the paged cache's entries refuse, before any launch: runs without a GPU (the pointers are never followed)."""
import ctypes

import pytest
import torch

import vlm_training_amd as V
from vlm_training_amd import _lib

FINE = dict(k=16, v=16, k_exp=16, v_exp=16, k_page=2 * 64 * 128, v_page=2 * 64 * 128, kx_page=2 * 64, vx_page=2 * 64, table=16, table_row=8, pages=4, page=64, table_pages=8, Hkv=2,
            D=128, kind=0)


def _args(**change):
    return ctypes.byref(_lib.CacheArgs(**{**FINE, **change}))


REFUSED = [(dict(kind=2), -1, b"kind"), (dict(D=12), -2, b"head_dim"), (dict(D=264), -2, b"head_dim"), (dict(D=0), -2, b"head_dim"), (dict(D=72, kind=1), -2, b"multiple of 16"),
           (dict(page=8), -2, b"pages of 8"), (dict(page=48), -2, b"pages of 48"), (dict(page=512), -2, b"pages of 512"), (dict(pages=0), -1, b"pages=0"), (dict(Hkv=0), -1, b"Hkv=0"),
           (dict(table_pages=0), -1, b"table_pages=0"), (dict(table_pages=(1 << 24) + 1, table_row=1 << 26), -2, b"2^30"), (dict(k_page=1 << 31), -2, b"4 GiB"), (dict(vx_page=1 << 32, kind=1), -2, b"4 GiB"), (dict(k=None), -1, b"null"), (dict(table=None), -1, b"null"),
           (dict(k_exp=None, kind=1), -1, b"null"), (dict(table_row=7), -1, b"table rows"), (dict(v=8), -1, b"16-byte"), (dict(k_page=2 * 64 * 128 + 4), -1, b"16-byte"),
           (dict(kx_page=136, kind=1), -1, b"16-byte"), (dict(v_page=2 * 64 * 128 - 8), -1, b"overlap"), (dict(vx_page=112, kind=1), -1, b"overlap")]


@pytest.mark.parametrize("change,code,text", REFUSED)
def test_caches(change, code, text):
    lib = _lib.load()
    calls = (lambda c: lib.dsa_cache_write(c, 16, 256, 128, 16, 256, 128, 16, 16, 8, 2, None), lambda c: lib.dsa_cache_read(c, 16, None, 8, 2, 16, 16, None),
             lambda c: lib.dsa_paged_attn(c, 16, 512, 128, 16, 16, 8, 2, 4, 1.0, 0, 0, 16, None, 16, 1 << 40, None))
    for call in calls:
        assert call(_args(**change)) == code and text in lib.dsa_last_error(), lib.dsa_last_error()
    assert lib.dsa_paged_attn_workspace_bytes(_args(**change), 8, 2, 4, 0, 0) == 0


def test_operands():
    lib = _lib.load()
    write = lambda k=16, tok=256, v=16, cu=16, lengths=16, T=8, N=2: lib.dsa_cache_write(_args(), k, tok, 128, v, 256, 128, cu, lengths, T, N, None)  # noqa: E731
    for change in (dict(k=None), dict(k=8), dict(tok=4), dict(v=None), dict(cu=None), dict(lengths=None), dict(T=-1), dict(N=0)):
        assert write(**change) == -1, change
    assert write(T=0) == 0 and lib.dsa_cache_write(None, 16, 256, 128, 16, 256, 128, 16, 16, 8, 2, None) == -1
    read = lambda cu=16, T=8, N=2, k=16, v=16: lib.dsa_cache_read(_args(), cu, None, T, N, k, v, None)  # noqa: E731
    for change in (dict(cu=None), dict(T=-1), dict(N=0), dict(k=None), dict(v=8)):
        assert read(**change) == -1, change
    assert read(T=0) == 0
    need = lib.dsa_paged_attn_workspace_bytes(_args(), 8, 2, 4, 0, 0)
    assert need > 0 and lib.dsa_paged_attn_workspace_bytes(_args(), 0, 2, 4, 0, 0) == 0 and lib.dsa_paged_attn_workspace_bytes(_args(), 8, 2, 4, 0, 100) == 0
    attn = lambda q=16, tok=512, cu=16, lengths=16, T=8, N=2, Hq=4, scale=1.0, new=0, longest=0, out=16, ws=16, n=need: lib.dsa_paged_attn(  # noqa: E731
        _args(), q, tok, 128, cu, lengths, T, N, Hq, scale, new, longest, out, None, ws, n, None)
    for change, code in ((dict(q=None), -1), (dict(q=8), -1), (dict(tok=12), -1), (dict(cu=None), -1), (dict(lengths=None), -1), (dict(T=-1), -1), (dict(N=0), -1), (dict(Hq=3), -1),
                         (dict(Hq=0), -1), (dict(Hq=34), -2), (dict(scale=float("inf")), -1), (dict(scale=float("nan")), -1), (dict(new=-1), -1), (dict(longest=-1), -1), (dict(out=None), -1),
                         (dict(out=8), -1), (dict(ws=None), -3), (dict(ws=8), -3), (dict(n=need - 1), -3)):
        assert attn(**change) == code, change
    assert attn(T=0) == 0
    for T, N, Hkv, new in ((1 << 30, 1 << 30, 2, 1), (1 << 26, 1 << 26, 2, 1), ((1 << 31) - 1, 1, 64, 0)):            # more blocks than a launch has room for
        many = _args(Hkv=Hkv, k_page=Hkv * 64 * 128, v_page=Hkv * 64 * 128)
        assert lib.dsa_paged_attn(many, 16, 512, 128, 16, 16, T, N, 2 * Hkv, 1.0, new, 0, 16, None, 16, 1 << 40, None) == -2 and b"too many" in lib.dsa_last_error()
        assert lib.dsa_paged_attn_workspace_bytes(many, T, N, 2 * Hkv, new, 0) == 0


def test_python_entries():
    """On the CPU every call ends at the device check; what comes in front of it is refused as what it is."""
    cache = V.KvCache.empty(2, 1, 64, page=16, device="cpu")
    assert cache.k.shape == (2, 1, 16, 64) and cache.k_scale is None
    small = V.KvCache.empty(2, 1, 64, page=16, dtype=torch.float8_e4m3fn, device="cpu")
    assert small.k.dtype == torch.float8_e4m3fn and small.k_scale.dtype == torch.float8_e8m0fnu and small.v_scale.shape == (2, 1, 16)
    with pytest.raises(ValueError):
        V.KvCache.empty(2, 1, 64, dtype=torch.float16, device="cpu")
    x, table, cu, lengths = torch.zeros(3, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32), torch.tensor([3], dtype=torch.int32)
    for call in (lambda: V.kv_cache_write(cache, x, x, table, cu, lengths), lambda: V.kv_cache_read(cache, table, cu, 3), lambda: V.paged_attn(x, cache, table, cu, lengths)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    grad = x.clone().requires_grad_(True)
    for call in (lambda: V.kv_cache_write(cache, grad, x, table, cu, lengths), lambda: V.paged_attn(grad, cache, table, cu, lengths)):
        with pytest.raises(ValueError, match="no backward"):
            call()


@pytest.mark.parametrize("page", [0, 8, 48, 512])
def test_empty_caches_of_other_pages(page):
    with pytest.raises(ValueError, match="page"):
        V.KvCache.empty(2, 1, 64, page=page, device="cpu")
