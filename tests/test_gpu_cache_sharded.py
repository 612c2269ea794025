"""The attention layers' serving form, head-sharded: with DTensor projections, and with the rows of some of the heads, as each rank of a tensor-parallel layer holds them."""
import copy

import pytest
import torch

import vlm_training_amd as V
from tests.test_gpu_cache_layer import _layer, _offsets, _run, _table, _tables
from tests.test_gpu_layers import _one_rank_cuda_mesh

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, E4 = torch.bfloat16, torch.float8_e4m3fn
KINDS = [(V.Qwen3VLTextAttention, 8, 4, 64, 64, 16, BF), (V.SelfAttention, 4, 2, 256, 64, 32, BF), (V.Qwen3VLTextAttention, 8, 2, 128, 128, 64, E4)]


def _inputs(lens, hidden):
    g = torch.Generator().manual_seed(1)
    return [torch.randn(n, hidden, generator=g).bfloat16().to(DEV) for n in lens]


def _extend(m, cache, table, lens, packed):
    if packed:
        return lambda x, cos, sin, cu, lengths, new: m.extend(x[None], cos, sin, cache, table, cu, lengths)[0]
    return lambda x, cos, sin, cu, lengths, new: m.extend(x, cos, sin, cache, table, cu, lengths, max_new=max(new), max_length=max(lens))


@pytest.mark.parametrize("cls,hq,hkv,dim,R,page,dtype", KINDS)
@pytest.mark.parametrize("packed", [False, True])
def test_dtensor_projections(cls, hq, hkv, dim, R, page, dtype, packed):
    """Column-parallel projections with DTensor outputs and a row-parallel o_proj on a mesh of one rank: the local shard is the whole, so outputs and caches are the plain layer's, bit for bit."""
    import torch.distributed as dist
    from torch.distributed.tensor import DTensor, Replicate
    from torch.distributed.tensor.parallel import ColwiseParallel, RowwiseParallel, SequenceParallel, parallelize_module
    print(cls.__name__, hq, hkv, dim, page, dtype, flush=True)
    lens, hidden = [150, 7, 61], hq * dim
    plain = _layer(cls, hidden, hq, hkv, dim, identity=False)
    table, pages = _table(lens, page)
    mesh, created = _one_rank_cuda_mesh()
    try:
        tp = copy.deepcopy(plain)
        parallelize_module(tp, mesh, {
            "q_proj": ColwiseParallel(use_local_output=False), "k_proj": ColwiseParallel(use_local_output=False), "v_proj": ColwiseParallel(use_local_output=False),
            "q_norm": SequenceParallel(sequence_dim=2), "k_norm": SequenceParallel(sequence_dim=2), "o_proj": RowwiseParallel(output_layouts=Replicate())}, src_data_rank=None)
        assert isinstance(tp.q_proj.weight, DTensor) and isinstance(tp.q_norm.weight, DTensor)
        xs, got = _inputs(lens, hidden), []
        for m in (plain, tp):
            cache = V.KvCache.empty(pages, hkv, dim, page=page, dtype=dtype)
            y = _run(_extend(m, cache, table, lens, packed), xs, lens, R)
            got.append((y.to_local() if isinstance(y, DTensor) else y, *(t.view(torch.uint8) for t in cache._parts() if t is not None)))
        assert all(torch.equal(a, b) for a, b in zip(*got)) and got[0][1].any()
    finally:
        if created:
            dist.destroy_process_group()


@pytest.mark.parametrize("cls,hq,hkv,dim,R,page,dtype", KINDS)
def test_a_rank_with_some_of_the_heads(cls, hq, hkv, dim, R, page, dtype):
    """Each of two ranks holds the projections' rows of its own heads and a cache of its own kv heads.  A projection of fewer columns may sum in another order, so that q, k and v may be off by
    a step of bf16: caches agree to 2^-6 of the largest value, what the ranks' outputs sum to has a cosine of 0.9999 with the whole layer's (the output's own rounding leaves 1 - 2^-17)."""
    print(cls.__name__, hq, hkv, dim, page, dtype, flush=True)
    lens, hidden, ranks = [150, 7, 61], hq * dim, 2
    whole = _layer(cls, hidden, hq, hkv, dim, identity=False)
    table, pages = _table(lens, page)
    xs = _inputs(lens, hidden)
    cache = V.KvCache.empty(pages, hkv, dim, page=page, dtype=dtype)
    want = _run(_extend(whole, cache, table, lens, False), xs, lens, R)
    rows = V.kv_cache_read(cache, table, _offsets(lens), sum(lens))
    total = 0
    for r in range(ranks):
        part = copy.deepcopy(whole)
        for name in ("q_proj", "k_proj", "v_proj"):
            lin = getattr(part, name)
            lin.weight = torch.nn.Parameter(lin.weight.chunk(ranks)[r].clone())
        part.o_proj.weight = torch.nn.Parameter(part.o_proj.weight.chunk(ranks, 1)[r].clone())
        own = V.KvCache.empty(pages, hkv // ranks, dim, page=page, dtype=dtype)
        total = total + _run(_extend(part, own, table, lens, False), xs, lens, R).double()
        for a, b in zip(V.kv_cache_read(own, table, _offsets(lens), sum(lens)), rows):
            b = b.chunk(ranks, 1)[r]
            # (8-bit: a value next to a border between two codes falls on either side, 2^-3 of it apart)
            assert ((a.float() - b.float()).abs() <= (2.0 ** -6 if dtype == BF else 2.0 ** -3) * b.float().abs().max()).all()
    cosine = torch.nn.functional.cosine_similarity(total.flatten(), want.double().flatten(), 0).item()
    assert cosine > (0.9999 if dtype == BF else 0.999), cosine
